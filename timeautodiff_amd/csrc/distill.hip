// Distillation loss of a student's logits against a teacher's top logits, and its gradient (gfx950).
//
//   q_k = softmax over the row's valid entries of value[r, k] / tau        (an index outside [0, V) is no entry)
//   p_j = softmax over the row of logits[r, j] / tau
//   loss[r] = w_r tau^2 sum_k q_k (ln q_k - ln p[index_k]),   dlogits[r, j] = grad_scale w_r tau (p_j - sum of the q_k with index_k = j)
//
// Statistics and sums in fp32, exponentials as 2^((x - max) log2(e) / tau) on the hardware's exp2 (the difference before the
// product: a row of the type's lowest values stays a row of zeros).  The loss is added up in the logits' own units, at half scale:
//
//   loss[r] = 2 w tau sum_k q_k ((value_k / 2 - max / 2) - (logit_k / 2 - max / 2) - tau / 2 (ln sum_teacher - ln sum_student))
//
// so that no part of it leaves fp32's range where the loss itself does not (an entry on a logit masked with the lowest value).
#include <limits.h>
#include <math.h>

#include "lanes.h"
#include "row_pieces.h"

namespace {

constexpr int MAX_K = 1024;
constexpr float LOWEST = -3.4028234663852886e38f;
constexpr float LN2 = 0.69314718055994531f;

struct Args {
  int64_t rows, V, ld, ld_t, ldd;
  int K;
  const int64_t* index;
  const float* value;
  const float* weight;
  float c, tau, grad_scale;         // c = log2(e) / tau
  float* loss;
};

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
// (x - largest) / 2, rounded once; finite for all finite x
__device__ __forceinline__ float half_from(float x, float largest) { return __builtin_fmaf(0.5f, x, -0.5f * largest); }

// ---------------------------------------------------------------- short rows: G lanes of a wave per row
// The row stays in registers (E logits a lane), statistics go across the G lanes by DPP, and the teacher's q reach their
// columns through LDS, which only the row's own lanes touch: its order within the wave is all the synchronisation.  An index
// that comes twice is seen by the entry whose mark at the column was overwritten; such entries add up all q of the index in
// order and write the same sum.  98304 x 48 float32, 8 entries: 11.3 us, 4.2 TB/s, and about as much instructions as HBM (q by
// 64-bit integer atomics and reductions by lane shuffles: 17 us).
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void distill_short_kernel(Args A, const T* logits, T* dlogits) {
  constexpr int R = 256 / G;                          // rows of a workgroup
  __shared__ uint32_t tgt[R][G * E];
  const int lane = threadIdx.x & (G - 1), slot = threadIdx.x / G;
  const int64_t r = (int64_t)blockIdx.x * R + slot;
  if (r >= A.rows) return;
  const int V = (int)A.V;
  const T* x = logits + r * A.ld;
  const int64_t* idx = A.index + r * A.ld_t;
  const float* val = A.value + r * A.ld_t;
  const auto entry = [&](int k) {                     // -1: none
    const int64_t i = idx[k];
    return (uint64_t)i < (uint64_t)V ? (int)i : -1;
  };
  // the lane's first entry stays in registers
  const int i0 = lane < A.K ? entry(lane) : -1;
  const float v0 = i0 >= 0 ? val[lane] : -INFINITY, x0 = i0 >= 0 ? (float)x[i0] : 0.f;
  const float w = A.weight ? A.weight[r] : 1.f;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = lane + e * G < V ? (float)x[lane + e * G] : -INFINITY;
  float m = LOWEST, tm = fmaxf(LOWEST, v0);
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
  for (int k = lane + G; k < A.K; k += G)
    if (entry(k) >= 0) tm = fmaxf(tm, val[k]);
  m = across<G, Max>(m);
  tm = across<G, Max>(tm);
  const float q0 = ex2((v0 - tm) * A.c);
  float z = 0.f, tz = q0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    v[e] = ex2((v[e] - m) * A.c);
    z += v[e];
  }
  for (int k = lane + G; k < A.K; k += G)
    if (entry(k) >= 0) tz += ex2((val[k] - tm) * A.c);
  z = across<G, Add>(z);
  tz = across<G, Add>(tz);
  const bool counts = w != 0.f && z != 0.f && tz != 0.f;
  const float itz = 1.f / tz, lz = 0.5f * A.tau * LN2 * (__log2f(tz) - __log2f(z));
  const auto term = [&](float q, float t, float s) { return q > 0.f ? q * (half_from(t, tm) - half_from(s, m) - lz) : 0.f; };
  float l = i0 >= 0 ? term(q0 * itz, v0, x0) : 0.f;
  for (int k = lane + G; k < A.K; k += G) {
    const int i = entry(k);
    if (i >= 0) l += term(ex2((val[k] - tm) * A.c) * itz, val[k], (float)x[i]);
  }
  l = across<G, Add>(l);
  if (lane == 0) A.loss[r] = counts ? 2.f * (w * A.tau * l) : 0.f;
  if (!dlogits) return;
  uint32_t* mine = tgt[slot];
  if (i0 >= 0) mine[i0] = lane;
  for (int k = lane + G; k < A.K; k += G)
    if (const int i = entry(k); i >= 0) mine[i] = k;
  lds_in_order();
  // an overwritten mark: the whole row takes the longer way
  int twice = i0 >= 0 && mine[i0] != (uint32_t)lane;
  for (int k = lane + G; k < A.K; k += G)
    if (const int i = entry(k); i >= 0) twice |= mine[i] != (uint32_t)k;
  twice = across<G, Max>(twice);
  lds_in_order();
#pragma unroll
  for (int e = 0; e < E; ++e) mine[lane + e * G] = 0;
  lds_in_order();
  for (int k = lane; k < A.K; k += G) {
    const int i = k == lane ? i0 : entry(k);
    if (i < 0) continue;
    float q = k == lane ? q0 * itz : ex2((val[k] - tm) * A.c) * itz;
    if (twice) {
      q = 0.f;
      for (int o = 0; o < A.K; ++o)
        if (entry(o) == i) q += ex2((val[o] - tm) * A.c) * itz;
    }
    mine[i] = __builtin_bit_cast(uint32_t, q);
  }
  lds_in_order();
  const float g = A.grad_scale * w * A.tau, iz = 1.f / z;
  T* d = dlogits + r * A.ldd;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = lane + e * G;
    if (j < V) d[j] = (T)(counts ? g * (v[e] * iz - __builtin_bit_cast(float, mine[j])) : 0.f);
  }
}

// ---------------------------------------------------------------- long rows: a workgroup per row
// Two passes over the row: maximum and sum in one (every thread rescales its sum when its maximum grows), then the gradient.
// A thread's first H pieces of 16 bytes stay in registers in between; the others are read again from the row's end backwards,
// where the caches still hold it, and the gradient goes past the caches.  4096 x 131072 bf16: 410 us, 4.9 TB/s of what it
// moves (nothing held 516, H = 8 / 16 / 20: 452 / 422 / 445, 24 at one workgroup a CU: 455; 1024 threads: 439; stores
// through the caches: 569); 512 x 32001 float32, the loss alone: 12.3 us, 4.8 TB/s.
template <int NW, bool MAX>
__device__ __forceinline__ void block_two(float& a, float& b, float (*s)[NW]) {      // largest, or sum, of two values at once
  a = MAX ? across<64, Max>(a) : wave_sum(a);
  b = MAX ? across<64, Max>(b) : wave_sum(b);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    s[0][threadIdx.x >> 6] = a;
    s[1][threadIdx.x >> 6] = b;
  }
  __syncthreads();
  a = s[0][0];
  b = s[1][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    a = MAX ? fmaxf(a, s[0][w]) : a + s[0][w];
    b = MAX ? fmaxf(b, s[1][w]) : b + s[1][w];
  }
}

template <typename T, int NT, int H>
__global__ __launch_bounds__(NT, NT == 512 ? 4 : 1) void distill_row_kernel(Args A, const T* logits, T* dlogits) {
  constexpr int VEC = RowPieces<T>::VEC, NW = NT / 64;
  typedef typename RowPieces<T>::pack pack;
  constexpr int KE = MAX_K / NT;                // the teacher's entries of a thread
  __shared__ float red[2][NW];
  __shared__ float q[MAX_K];
  __shared__ int at[MAX_K];
  const int tid = threadIdx.x, K = A.K;
  const int64_t r = blockIdx.x, V = A.V;
  const T* x = logits + r * A.ld;
  T* d = dlogits ? dlogits + r * A.ldd : nullptr;
  // `head` elements up to a 16-byte boundary, np whole pieces from there, and what is left: head and rest one by one, by the
  // first threads.  (The gradient's rows may lie differently: its stores need the alignment of an element only.)
  const int head = (int)(-((uintptr_t)x / sizeof(T)) & (VEC - 1));
  const int64_t np = (V - head) / VEC;
  const int edge = (int)(V - np * VEC);
  const int64_t at_edge = tid < head ? tid : V - edge + tid;
  const auto piece = [&](int64_t i) { return *reinterpret_cast<const pack*>(x + head + i * VEC); };
  const float w = A.weight ? A.weight[r] : 1.f;
  float m = LOWEST, z = 0.f, tm = LOWEST, tz = 0.f;
  // the entries and the student's logits at them, asked for before anything waits
  int mine[KE];
  float val[KE], xv[KE];
#pragma unroll
  for (int n = 0; n < KE; ++n) {
    const int k = tid + n * NT;
    mine[n] = -1;
    val[n] = xv[n] = 0.f;
    if (k < K) {
      const int64_t i = A.index[r * A.ld_t + k];
      mine[n] = (uint64_t)i < (uint64_t)V ? (int)i : -1;
      val[n] = A.value[r * A.ld_t + k];
      if (mine[n] >= 0) xv[n] = (float)x[mine[n]];
    }
  }
  const auto add = [&](const pack& p) {
    float b = m;
#pragma unroll
    for (int e = 0; e < VEC; ++e) b = fmaxf(b, (float)p[e]);
    float s = z * ex2((m - b) * A.c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += ex2(((float)p[e] - b) * A.c);
    m = b;
    z = s;
  };
  pack held[H];
  float last = -INFINITY;
  if (w != 0.f) {
#pragma unroll
    for (int k = 0; k < H; ++k)
      if (tid + k * NT < np) held[k] = piece(tid + k * NT);
    if (tid < edge) last = (float)x[at_edge];
#pragma unroll
    for (int k = 0; k < H; ++k)
      if (tid + k * NT < np) add(held[k]);
#pragma unroll 4
    for (int64_t i = tid + H * NT; i < np; i += NT) add(piece(i));
    if (tid < edge) {
      const float b = fmaxf(m, last);
      z = z * ex2((m - b) * A.c) + ex2((last - b) * A.c);
      m = b;
    }
  }
#pragma unroll
  for (int n = 0; n < KE; ++n)
    if (mine[n] >= 0) tm = fmaxf(tm, val[n]);
  const float own = m;
  block_two<NW, true>(m, tm, red);
  z *= ex2((own - m) * A.c);
  float p[KE], qn[KE];
#pragma unroll
  for (int n = 0; n < KE; ++n) {
    qn[n] = mine[n] >= 0 ? ex2((val[n] - tm) * A.c) : 0.f;
    tz += qn[n];
  }
  block_two<NW, false>(z, tz, red);
  if (w == 0.f || z == 0.f || tz == 0.f) {          // the row counts nothing
    if (tid == 0) A.loss[r] = 0.f;
    if (d)
      for (int64_t j = tid; j < V; j += NT) d[j] = (T)0.f;
    return;
  }
  const float itz = 1.f / tz, iz = 1.f / z, lz = 0.5f * A.tau * LN2 * (__log2f(tz) - __log2f(z)), g = A.grad_scale * w * A.tau;
  float l = 0.f, unused = 0.f;
#pragma unroll
  for (int n = 0; n < KE; ++n) {
    p[n] = ex2((xv[n] - m) * A.c) * iz;
    qn[n] *= itz;
    if (qn[n] > 0.f) l += qn[n] * (half_from(val[n], tm) - half_from(xv[n], m) - lz);
    if (tid + n * NT < K) {
      q[tid + n * NT] = qn[n];
      at[tid + n * NT] = mine[n];
    }
  }
  block_two<NW, false>(l, unused, red);
  if (tid == 0) A.loss[r] = 2.f * (w * A.tau * l);
  if (!d) return;
  const float gz = g * iz;
  const auto put = [&](int64_t i, const pack& p) {
    pack o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (T)(gz * ex2(((float)p[e] - m) * A.c));
    __builtin_nontemporal_store(o, reinterpret_cast<pack*>(d + head + i * VEC));
  };
#pragma unroll 4
  for (int64_t i = tid < np ? (np - 1 - tid) / NT * NT + tid : -1; i >= H * NT; i -= NT) put(i, piece(i));
#pragma unroll
  for (int k = 0; k < H; ++k)
    if (tid + k * NT < np) put(tid + k * NT, held[k]);
  if (tid < edge) d[at_edge] = (T)(gz * ex2((last - m) * A.c));
  __syncthreads();
#pragma unroll
  for (int n = 0; n < KE; ++n) {
    if (mine[n] < 0) continue;
    float sum = 0.f;
    bool first = true;
    for (int o = 0; o < K; ++o) {
      if (at[o] != mine[n]) continue;
      if (o < tid + n * NT) first = false;
      sum += q[o];
    }
    if (first) d[mine[n]] = (T)(g * (p[n] - sum));
  }
}

template <typename T>
int launch_distill(const Args& A, const T* x, T* d, hipStream_t s) {
  // 4, 16 or 64 lanes a row, so that a lane has at most 16 logits; then workgroups of 256 threads, which hold 8192 bf16 or 4096
  // float32 logits (16384 x 5000 bf16, K = 64: 103 us; 512 threads: 119); beyond 16384 logits of 512 threads, in bf16 with 8
  // pieces each as long as these hold the row (8192 x 32001, K = 64: 229 us; with 16: 242), then with 16 (4096 x 50001 bf16: 177;
  // with 8: 187, 24: 185; 4096 x 32001 float32: 217; with 8: 259)
  constexpr int MIDDLE = sizeof(T) == 2 ? 8 : 16;
#define SHORT_(G, E) hipLaunchKernelGGL((distill_short_kernel<T, G, E>), dim3((unsigned)cdiv64(A.rows, 256 / G)), dim3(256), 0, s, A, x, d)
#define ROW_(NT, H) hipLaunchKernelGGL((distill_row_kernel<T, NT, H>), dim3((unsigned)A.rows), dim3(NT), 0, s, A, x, d)
  if (A.V <= 16) SHORT_(4, 4);
  else if (A.V <= 32) SHORT_(16, 2);
  else if (A.V <= 48) SHORT_(16, 3);
  else if (A.V <= 64) SHORT_(16, 4);
  else if (A.V <= 128) SHORT_(16, 8);
  else if (A.V <= 256) SHORT_(64, 4);
  else if (A.V <= 512) SHORT_(64, 8);
  else if (A.V <= 1024) SHORT_(64, 16);
  else if (A.V <= 16384) ROW_(256, 4);
  else if (A.V <= 32768) ROW_(512, MIDDLE);
  else ROW_(512, 16);
#undef SHORT_
#undef ROW_
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}

}  // namespace

extern "C" int tad_distill_loss(int64_t rows, int64_t V, int K, const void* logits, int dtype, int64_t ld, const int64_t* index, const float* value,
                                int64_t ld_t, float tau, const float* row_weight, float grad_scale, float* loss_rows, void* dlogits, int64_t ldd,
                                tad_stream_t stream) {
  TAD_CHECK(rows >= 0 && V >= 1 && V <= INT_MAX && K >= 1 && K <= MAX_K, "tad_distill_loss: bad sizes (at most %d entries a row)", MAX_K);
  TAD_CHECK(dtype == TAD_F32 || dtype == TAD_BF16, "tad_distill_loss: bad element type");
  TAD_CHECK(ld >= V && ld_t >= K && (!dlogits || ldd >= V), "tad_distill_loss: bad leading dimension");
  TAD_CHECK(tau >= 1e-18f && tau <= 1e18f, "tad_distill_loss: the temperature has to lie between 1e-18 and 1e18");
  if (rows == 0) return TAD_OK;
  TAD_CHECK(logits && index && value && loss_rows, "tad_distill_loss: null pointer");
  TAD_CHECK(dlogits != logits || ldd == ld, "tad_distill_loss: a gradient in the logits' place needs their row stride");
  // at most 2^22 rows a launch: a grid holds fewer than 2^32 threads
  const int64_t step = (int64_t)1 << 22;
  for (int64_t r = 0; r < rows; r += step) {
    const Args A = {rows - r < step ? rows - r : step, V, ld, ld_t, ldd, K, index + r * ld_t, value + r * ld_t, row_weight ? row_weight + r : nullptr,
                    (float)(1.4426950408889634074 / (double)tau), tau, grad_scale, loss_rows + r};
    const int64_t x = r * ld, d = r * ldd;
    const int rc = dtype == TAD_F32
                       ? launch_distill<float>(A, (const float*)logits + x, dlogits ? (float*)dlogits + d : nullptr, (hipStream_t)stream)
                       : launch_distill<bf16_t>(A, (const bf16_t*)logits + x, dlogits ? (bf16_t*)dlogits + d : nullptr, (hipStream_t)stream);
    if (rc != TAD_OK) return rc;
  }
  return TAD_OK;
}
