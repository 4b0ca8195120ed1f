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
template <int VEC> struct Pack<float, VEC> { typedef __attribute__((ext_vector_type(VEC))) float type; };
template <int VEC> struct Pack<bf16_t, VEC> { typedef __attribute__((ext_vector_type(VEC))) __bf16 type; };
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

// ---------------------------------------------------------------- forward
// L lanes (a power of two, at most a wave) walk the columns of one row; a wave holds 64 / L rows side by side and EF_U of
// them one after another, whose loads are all issued before the first is used.
constexpr int EF_U = 4;

template <typename TI, typename TO, int VEC>
__global__ __launch_bounds__(256) void token_embed_fwd_kernel(int64_t n, int nv, int lanes_log2, int64_t vocab, const int64_t* __restrict__ tok,
                                                              int64_t tstride, float scale, const TI* __restrict__ table, int64_t ldt,
                                                              TO* __restrict__ out, int64_t ldo) {
  const int L = 1 << lanes_log2;
  const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lanes_log2;     // EF_U rows each
  const int64_t ngroups = ((int64_t)gridDim.x * 256) >> lanes_log2;
  const int lane = threadIdx.x & (L - 1);
  int64_t row[EF_U], t[EF_U];
#pragma unroll
  for (int u = 0; u < EF_U; ++u) {
    row[u] = group + u * ngroups;
    t[u] = row[u] < n ? tok[row[u] * tstride] : -1;
  }
  for (int c = lane; c < nv; c += L) {
    float v[EF_U][VEC];
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
      if ((uint64_t)t[u] < (uint64_t)vocab) load_pack<TI, VEC>(table + t[u] * ldt + (int64_t)c * VEC, v[u]);
    }
#pragma unroll
    for (int u = 0; u < EF_U; ++u) {
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
// key = token << 32 | position: all keys differ, and their order is the tokens' with equal ones by position.  Padding gets
// the token `vocab`, behind every other.  A workgroup sorts a tile in LDS; tiles are merged by rank: a key's place among
// the merged lists is its place in its own list plus, for every other list, how many of that list's keys are less (a
// binary search): no workgroup waits for another, and no distribution of tokens is worse than another.
constexpr int TILE = 4096;
constexpr int FANIN = 32;     // lists merged by one launch

__global__ __launch_bounds__(1024) void sort_tile_kernel(int64_t n, int64_t vocab, const int64_t* __restrict__ tok, int64_t tstride,
                                                         u64* __restrict__ keys) {
  __shared__ u64 s[TILE];
  const int64_t base = (int64_t)blockIdx.x * TILE;
  const int m = (int)(n - base < TILE ? n - base : TILE);
  int P = 64;
  while (P < m) P <<= 1;
  for (int i = threadIdx.x; i < P; i += 1024) {
    u64 k = ~0ull;
    if (i < m) {
      const int64_t t = tok[(base + i) * tstride];
      k = ((u64)((uint64_t)t < (uint64_t)vocab ? t : vocab) << 32) | (u64)(base + i);
    }
    s[i] = k;
  }
  __syncthreads();
  for (int size = 2; size <= P; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = threadIdx.x; i < P / 2; i += 1024) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const u64 a = s[lo], b = s[hi];
        if ((a > b) == ((lo & size) == 0)) { s[lo] = b; s[hi] = a; }
      }
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < m; i += 1024) keys[base + i] = s[i];
}

// lists of `len` sorted keys each (the last one shorter), FANIN of them merged into one
__global__ __launch_bounds__(256) void merge_rank_kernel(int64_t n, int64_t len, const u64* __restrict__ in, u64* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const u64 key = in[i];
  const int64_t mine = i / len, first = mine / FANIN * FANIN;
  int64_t rank = i - mine * len;
  for (int64_t l = first; l < first + FANIN && l * len < n; ++l) {
    if (l == mine) continue;
    const u64* p = in + l * len;
    int64_t lo = 0, hi = n - l * len < len ? n - l * len : len;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (p[mid] < key) lo = mid + 1; else hi = mid;
    }
    rank += lo;
  }
  out[first * len + rank] = key;
}

// ---------------------------------------------------------------- sums over the sorted tokens
// A wave adds the rows of `S` neighbouring sorted positions, 64 * VEC columns of them.  A run of equal tokens that lies
// inside the chunk is a finished row of dtable; what reaches over an edge goes to the workspace (slot 0: the run that came
// in from the left; slot 1: one that begins here and goes on) and is added up by the launch behind.
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
  store_pack<float, VEC>(dt, v);
}

constexpr int ZROWS = 16;     // rows of the table a wave of the zero part looks after

template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_sum_kernel(int64_t n, int D, int64_t vocab, int S, int64_t nchunks, int ctiles, float scale,
                                                             int accumulate, const u64* __restrict__ keys, const T* __restrict__ dout, int64_t ldd,
                                                             float* __restrict__ dtable, int64_t ldg, float* __restrict__ part) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t nsum = nchunks * ctiles;
  if (w >= nsum) {
    // rows that no token names are zero (overwriting mode): a lane looks one row up in the sorted keys
    const int64_t v0 = (w - nsum) * ZROWS;
    if (accumulate || v0 >= vocab) return;
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
        store_pack<float, VEC>(row + c, z);
      }
    }
    return;
  }
  const int64_t chunk = w / ctiles;
  const int c = (int)(w - chunk * ctiles) * 64 * VEC + lane * VEC;
  const int64_t a = chunk * S, b = a + S < n ? a + S : n;
  const bool on = c < D;
  const uint32_t before = a > 0 ? (uint32_t)(keys[a - 1] >> 32) : UINT_MAX;
  const uint32_t after = b < n ? (uint32_t)(keys[b] >> 32) : UINT_MAX;
  float acc[VEC] = {};
  uint32_t cur = (uint32_t)(keys[a] >> 32);
  bool from_left = cur == before;
  for (int64_t j = a; j < b; ++j) {
    const u64 k = keys[j];
    const uint32_t t = (uint32_t)(k >> 32);
    if (t >= (uint64_t)vocab) break;                     // padding lies behind everything else
    if (on) {
      float v[VEC];
      load_pack<T, VEC>(dout + (int64_t)(uint32_t)k * ldd + c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += v[i];
    }
    const uint32_t next = j + 1 < b ? (uint32_t)(keys[j + 1] >> 32) : after;
    if (next != t || j + 1 == b) {
      if (on) {
        if (from_left) store_pack<float, VEC>(part + (2 * chunk) * D + c, acc);
        else if (next == t) store_pack<float, VEC>(part + (2 * chunk + 1) * D + c, acc);
        else put_row<VEC>(dtable + (int64_t)t * ldg + c, acc, scale, accumulate);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
      from_left = false;
    }
  }
}

// Runs that reach over the edges of chunks: a workgroup for each chunk in which one begins (the others leave at once) and
// each 64 columns; its waves add every fourth part, and the four sums are added in order.
__global__ __launch_bounds__(256) void embed_grad_join_kernel(int64_t n, int D, int64_t vocab, int S, int ctiles, float scale, int accumulate,
                                                              const u64* __restrict__ keys, const float* __restrict__ part,
                                                              float* __restrict__ dtable, int64_t ldg) {
  const int64_t chunk = blockIdx.x / ctiles;
  const int c = (int)(blockIdx.x - chunk * ctiles) * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  const int64_t a = chunk * S, b = a + S;
  if (b >= n) return;
  const uint32_t t = (uint32_t)(keys[b - 1] >> 32);
  if (t >= (uint64_t)vocab || (uint32_t)(keys[b] >> 32) != t) return;
  if (a > 0 && (uint32_t)(keys[a - 1] >> 32) == t) return;      // began in an earlier chunk
  const u64 end = (u64)(t + 1) << 32;
  int64_t lo = b, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < end) lo = mid + 1; else hi = mid;
  }
  const int64_t last = (lo - 1) / S;                             // the chunk in which the run ends
  float acc = 0.f;
  if (c < D) {
    if (wave == 0) acc = part[(2 * chunk + 1) * D + c];
    for (int64_t k = chunk + 1 + wave; k <= last; k += 4) acc += part[(2 * k) * D + c];
  }
  __shared__ float s[4][64];
  s[wave][threadIdx.x & 63] = acc;
  __syncthreads();
  if (wave == 0 && c < D) {
    const float v = (((s[0][threadIdx.x] + s[1][threadIdx.x]) + s[2][threadIdx.x]) + s[3][threadIdx.x]) * scale;
    float* dt = dtable + (int64_t)t * ldg + c;
    *dt = accumulate ? *dt + v : v;
  }
}

// ---------------------------------------------------------------- host side
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// How the gradient is cut: S positions a wave, VEC columns a lane.
struct GradPlan {
  int vec, S, ctiles;
  int64_t nchunks;
};
GradPlan grad_plan(int64_t n, int D, int dtype, bool wide) {
  GradPlan g;
  const int most = dtype == TAD_BF16 ? 8 : 4;
  g.vec = 1;
  if (wide)
    while (g.vec < most && D >= 128 * g.vec) g.vec *= 2;
  g.ctiles = (int)cdiv64(D, 64 * g.vec);
  g.S = 64;
  while (g.S > 8 && cdiv64(n, g.S) * g.ctiles < 4096) g.S /= 2;
  g.nchunks = cdiv64(n, g.S);
  return g;
}

template <typename TI, typename TO>
int launch_fwd(int64_t n, int D, int64_t vocab, const int64_t* tok, int64_t tstride, float scale, const void* table, int64_t ldt, void* out,
               int64_t ldo, hipStream_t s) {
  constexpr int V = sizeof(TI) == 2 && sizeof(TO) == 2 ? 8 : 4;
  const bool wide = D % V == 0 && ldt % V == 0 && ldo % V == 0 && aligned16(table) && aligned16(out);
  const int nv = wide ? D / V : D;
  int ll = 0;
  while (ll < 6 && (1 << ll) < nv) ++ll;
  const int64_t groups = cdiv64(n, EF_U), grid = cdiv64(groups << ll, 256);
  TAD_CHECK(grid <= INT_MAX, "tad_token_embed_fwd: too many tokens");
  if (wide)
    hipLaunchKernelGGL((token_embed_fwd_kernel<TI, TO, V>), dim3((unsigned)grid), dim3(256), 0, s, n, nv, ll, vocab, tok, tstride, scale,
                       (const TI*)table, ldt, (TO*)out, ldo);
  else
    hipLaunchKernelGGL((token_embed_fwd_kernel<TI, TO, 1>), dim3((unsigned)grid), dim3(256), 0, s, n, nv, ll, vocab, tok, tstride, scale,
                       (const TI*)table, ldt, (TO*)out, ldo);
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}

template <typename T, int VEC>
void launch_sum(const GradPlan& g, int64_t n, int D, int64_t vocab, float scale, int accumulate, const u64* keys, const void* dout, int64_t ldd,
                float* dtable, int64_t ldg, float* part, hipStream_t s) {
  const int64_t waves = g.nchunks * g.ctiles + (accumulate ? 0 : cdiv64(vocab, ZROWS));
  hipLaunchKernelGGL((embed_grad_sum_kernel<T, VEC>), dim3((unsigned)cdiv64(waves, 4)), dim3(256), 0, s, n, D, vocab, g.S, g.nchunks, g.ctiles,
                     scale, accumulate, keys, (const T*)dout, ldd, dtable, ldg, part);
}

}  // namespace

extern "C" int tad_token_embed_fwd(int64_t n, int D, int64_t vocab, const int64_t* tokens, int64_t tok_stride, float scale, const void* table,
                                   int table_dtype, int64_t ld_table, void* out, int out_dtype, int64_t ldo, tad_stream_t stream) {
  TAD_CHECK(n >= 0 && D >= 1 && vocab >= 0, "tad_token_embed_fwd: bad sizes");
  TAD_CHECK((table_dtype == TAD_F32 || table_dtype == TAD_BF16) && (out_dtype == TAD_F32 || out_dtype == TAD_BF16), "tad_token_embed_fwd: bad element type");
  TAD_CHECK(ld_table >= D && ldo >= D && tok_stride >= 0, "tad_token_embed_fwd: bad leading dimension");
  if (n == 0) return TAD_OK;
  TAD_CHECK(tokens && out && (table || vocab == 0), "tad_token_embed_fwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (table_dtype == TAD_F32)
    return out_dtype == TAD_F32 ? launch_fwd<float, float>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s)
                                : launch_fwd<float, bf16_t>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s);
  return out_dtype == TAD_F32 ? launch_fwd<bf16_t, float>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s)
                              : launch_fwd<bf16_t, bf16_t>(n, D, vocab, tokens, tok_stride, scale, table, ld_table, out, ldo, s);
}

// keys twice (the lists and their merge), then the parts of runs over edges
extern "C" int64_t tad_token_embed_bwd_workspace_bytes(int64_t n, int D) {
  if (n <= 0 || D < 1) return 0;
  // the parts of the finest cut that any alignment or type of dout leads to
  int64_t part = 0;
  for (int dt = TAD_F32; dt <= TAD_BF16; ++dt)
    for (int wide = 0; wide < 2; ++wide) {
      const GradPlan g = grad_plan(n, D, dt, wide);
      if (2 * g.nchunks * D > part) part = 2 * g.nchunks * D;
    }
  return 2 * ((n * 8 + 15) / 16 * 16) + part * 4;
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
  const bool wide = ld_dtable % 4 == 0 && D % (dout_dtype == TAD_BF16 ? 8 : 4) == 0 && ld_dout % (dout_dtype == TAD_BF16 ? 8 : 4) == 0 &&
                    aligned16(dout) && aligned16(dtable);
  const GradPlan g = grad_plan(n, D, dout_dtype, wide);
  const int64_t kb = (n * 8 + 15) / 16 * 16;
  TAD_CHECK(workspace && aligned16(workspace) && workspace_bytes >= 2 * kb + 2 * g.nchunks * D * 4,
            "tad_token_embed_bwd: workspace of %lld bytes, 16-byte aligned, needed", (long long)tad_token_embed_bwd_workspace_bytes(n, D));
  TAD_CHECK((g.nchunks * g.ctiles + cdiv64(vocab, ZROWS)) / 4 < INT_MAX && g.nchunks * cdiv64(D, 64) < INT_MAX, "tad_token_embed_bwd: too many tokens");
  u64* a = (u64*)workspace;
  u64* b = (u64*)((char*)workspace + kb);
  float* part = (float*)((char*)workspace + 2 * kb);
  hipLaunchKernelGGL(sort_tile_kernel, dim3((unsigned)cdiv64(n, TILE)), dim3(1024), 0, s, n, vocab, tokens, tok_stride, a);
  TAD_LAUNCH_CHECK();
  for (int64_t len = TILE; len < n; len *= FANIN) {
    hipLaunchKernelGGL(merge_rank_kernel, dim3((unsigned)cdiv64(n, 256)), dim3(256), 0, s, n, len, a, b);
    TAD_LAUNCH_CHECK();
    u64* t = a; a = b; b = t;
  }
#define SUM_(T, V) launch_sum<T, V>(g, n, D, vocab, scale, accumulate, a, dout, ld_dout, dtable, ld_dtable, part, s)
  if (dout_dtype == TAD_BF16) {
    if (g.vec == 8) SUM_(bf16_t, 8); else if (g.vec == 4) SUM_(bf16_t, 4); else if (g.vec == 2) SUM_(bf16_t, 2); else SUM_(bf16_t, 1);
  } else {
    if (g.vec == 4) SUM_(float, 4); else if (g.vec == 2) SUM_(float, 2); else SUM_(float, 1);
  }
#undef SUM_
  TAD_LAUNCH_CHECK();
  if (g.nchunks > 1) {
    const int ct = (int)cdiv64(D, 64);
    hipLaunchKernelGGL(embed_grad_join_kernel, dim3((unsigned)(g.nchunks * ct)), dim3(256), 0, s, n, D, vocab, g.S, ct, scale, accumulate, a, part,
                       dtable, ld_dtable);
    TAD_LAUNCH_CHECK();
  }
  tad_note_kernel("embed_grad_sum_kernel");
  return TAD_OK;
}
