// Distillation loss of a student's logits against a teacher's top logits, and its gradient (gfx950).
//
//   q_k = softmax over the row's valid entries of value[r, k] / tau        (an index outside [0, V) is no entry)
//   p_j = softmax over the row of logits[r, j] / tau
//   loss[r] = w_r tau^2 sum_k q_k (ln q_k - ln p[index_k]),   dlogits[r, j] = grad_scale w_r tau (p_j - sum of the q_k with index_k = j)
//
// Statistics and sums in fp32, exponentials as 2^((x - max) log2(e) / tau) on the hardware's exp2 (the difference before the
// product: a row of the type's lowest values stays a row of zeros).
#include <limits.h>
#include <math.h>

#include "row_pieces.h"

namespace {

typedef unsigned long long u64;

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

// ---------------------------------------------------------------- short rows: G lanes of a wave per row
// The row stays in registers (E logits a lane), statistics go across the G lanes; the teacher's q are laid into LDS by their
// indices, as multiples of 2^-60 in 64-bit integers, so that an index that comes twice has the same sum in any order.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

template <typename T, int G, int E>
__global__ __launch_bounds__(256) void distill_short_kernel(Args A, const T* logits, T* dlogits) {
  constexpr int R = 256 / G;                          // rows of a workgroup
  __shared__ u64 tgt[R][G * E];
  const int lane = threadIdx.x & (G - 1), slot = threadIdx.x / G;
  const int64_t r = (int64_t)blockIdx.x * R + slot;
  const bool live = r < A.rows;
  const int V = (int)A.V;
  const T* x = logits + (live ? r : 0) * A.ld;
  const float w = live ? (A.weight ? A.weight[r] : 1.f) : 0.f;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = lane + e * G;
    v[e] = j < V ? (float)x[j] : -INFINITY;
    tgt[slot][j] = 0;
  }
  float m = LOWEST;
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
  m = group_max<G>(m);
  float z = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    v[e] = ex2((v[e] - m) * A.c);
    z += v[e];
  }
  z = group_sum<G>(z);
  const int64_t* idx = A.index + (live ? r : 0) * A.ld_t;
  const float* val = A.value + (live ? r : 0) * A.ld_t;
  float tm = LOWEST;
  for (int k = lane; k < A.K; k += G)
    if ((uint64_t)idx[k] < (uint64_t)V) tm = fmaxf(tm, val[k]);
  tm = group_max<G>(tm);
  float tz = 0.f;
  for (int k = lane; k < A.K; k += G)
    if ((uint64_t)idx[k] < (uint64_t)V) tz += ex2((val[k] - tm) * A.c);
  tz = group_sum<G>(tz);
  const bool counts = w != 0.f && z != 0.f && tz != 0.f;
  const float itz = 1.f / tz, l2 = __log2f(tz) - __log2f(z);
  float l = 0.f;
  if (dlogits) __syncthreads();
  for (int k = lane; k < A.K; k += G) {
    const int64_t i = idx[k];
    if ((uint64_t)i >= (uint64_t)V) continue;
    const float a = (val[k] - tm) * A.c, q = ex2(a) * itz;
    if (!(q > 0.f)) continue;
    l += q * (a - ((float)x[i] - m) * A.c - l2);
    if (dlogits) atomicAdd(&tgt[slot][i], (u64)((double)q * 1152921504606846976.0));
  }
  l = group_sum<G>(l);
  if (lane == 0 && live) A.loss[r] = counts ? w * A.tau * A.tau * (l * LN2) : 0.f;
  if (!dlogits) return;
  __syncthreads();
  if (!live) return;
  const float g = A.grad_scale * w * A.tau, iz = 1.f / z;
  T* d = dlogits + r * A.ldd;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = lane + e * G;
    if (j < V) {
      const u64 q = tgt[slot][j];
      float t = 0.f;
      if (q) t = (float)((double)q * (1.0 / 1152921504606846976.0));
      d[j] = (T)(counts ? g * (v[e] * iz - t) : 0.f);
    }
  }
}

// ---------------------------------------------------------------- long rows: a workgroup per row
// Two passes over the row: maximum and sum in one (every thread rescales its sum when its maximum grows), then the gradient,
// from the row's end backwards, where the caches still hold it.
template <int NW>
__device__ __forceinline__ float block_sum(float v, float* s) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) t += s[w];
  return t;
}
template <int NW>
__device__ __forceinline__ float block_max(float v, float* s) {
  v = group_max<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = s[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) t = fmaxf(t, s[w]);
  return t;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_row_kernel(Args A, const T* logits, T* dlogits) {
  constexpr int VEC = RowPieces<T>::VEC, NW = NT / 64;
  typedef typename RowPieces<T>::pack pack;
  __shared__ float red[NW];
  __shared__ float q[MAX_K];
  __shared__ int at[MAX_K];
  const int tid = threadIdx.x, K = A.K;
  const int64_t r = blockIdx.x, V = A.V;
  const T* x = logits + r * A.ld;
  T* d = dlogits ? dlogits + r * A.ldd : nullptr;
  const RowPieces<T> row(x, V);
  const float w = A.weight ? A.weight[r] : 1.f;
  float m = LOWEST, z = 0.f;
  if (w != 0.f) {
#pragma unroll 4
    for (int64_t i = tid; i < row.np; i += NT) {
      float v[VEC];
      row.load(i, v);
      float b = m;
#pragma unroll
      for (int e = 0; e < VEC; ++e) b = fmaxf(b, v[e]);
      float s = z * ex2((m - b) * A.c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += ex2((v[e] - b) * A.c);
      m = b;
      z = s;
    }
  }
  const float mine = m;
  m = block_max<NW>(m, red);
  z = block_sum<NW>(z * ex2((mine - m) * A.c), red);
  float tz = 0.f, tm = LOWEST;
  if (w != 0.f && z != 0.f) {
    for (int k = tid; k < K; k += NT) {
      const int64_t i = A.index[r * A.ld_t + k];
      at[k] = (uint64_t)i < (uint64_t)V ? (int)i : -1;
      if (at[k] >= 0) tm = fmaxf(tm, A.value[r * A.ld_t + k]);
    }
    tm = block_max<NW>(tm, red);
    for (int k = tid; k < K; k += NT) {
      q[k] = at[k] >= 0 ? ex2((A.value[r * A.ld_t + k] - tm) * A.c) : 0.f;
      tz += q[k];
    }
    tz = block_sum<NW>(tz, red);
  }
  if (tz == 0.f) {          // the row counts nothing: weight 0, no student logit or no entry above -inf
    if (tid == 0) A.loss[r] = 0.f;
    if (d)
      for (int64_t j = tid; j < V; j += NT) d[j] = (T)0.f;
    return;
  }
  const float itz = 1.f / tz, iz = 1.f / z, l2 = __log2f(tz) - __log2f(z), g = A.grad_scale * w * A.tau;
  float l = 0.f;
  float px[MAX_K / NT > 0 ? MAX_K / NT : 1];             // the student's p at this thread's entries, before the row may be overwritten
#pragma unroll
  for (int n = 0; n < (MAX_K / NT > 0 ? MAX_K / NT : 1); ++n) {
    const int k = tid + n * NT;
    px[n] = 0.f;
    if (k >= K) continue;
    q[k] *= itz;
    if (at[k] < 0) continue;
    const float b = ((float)x[at[k]] - m) * A.c;
    px[n] = ex2(b) * iz;
    if (q[k] > 0.f) l += q[k] * ((A.value[r * A.ld_t + k] - tm) * A.c - b - l2);
  }
  l = block_sum<NW>(l, red);
  if (tid == 0) A.loss[r] = w * A.tau * A.tau * (l * LN2);
  if (!d) return;
  __syncthreads();
  const float gz = g * iz;
  const bool together = (((uintptr_t)d ^ (uintptr_t)x) & 15) == 0;
  const int64_t last = tid < row.np ? (row.np - 1 - tid) / NT * NT + tid : -1;
#pragma unroll 4
  for (int64_t i = last; i >= 0; i -= NT) {
    float v[VEC];
    row.load(i, v);
    pack o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (T)(gz * ex2((v[e] - m) * A.c));
    const int64_t j = row.first(i);
    if (together && j >= 0 && j + VEC <= V) {
      *reinterpret_cast<pack*>(d + j) = o;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (j + e >= 0 && j + e < V) d[j + e] = o[e];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < (MAX_K / NT > 0 ? MAX_K / NT : 1); ++n) {
    const int k = tid + n * NT;
    if (k >= K || at[k] < 0) continue;
    float s = 0.f;
    bool first = true;
    for (int o = 0; o < K; ++o) {
      if (at[o] != at[k]) continue;
      if (o < k) first = false;
      s += q[o];
    }
    if (first) d[at[k]] = (T)(g * (px[n] - s));
  }
}

template <typename T>
int launch_distill(const Args& A, const T* x, T* d, hipStream_t s) {
#define SHORT_(G, E) hipLaunchKernelGGL((distill_short_kernel<T, G, E>), dim3((unsigned)cdiv64(A.rows, 256 / G)), dim3(256), 0, s, A, x, d)
#define ROW_(NT) hipLaunchKernelGGL((distill_row_kernel<T, NT>), dim3((unsigned)A.rows), dim3(NT), 0, s, A, x, d)
  if (A.V <= 32) SHORT_(8, 4);
  else if (A.V <= 64) SHORT_(16, 4);
  else if (A.V <= 128) SHORT_(16, 8);
  else if (A.V <= 1024) SHORT_(64, 16);
  else if (A.V <= 16384) ROW_(256);
  else ROW_(1024);
#undef SHORT_
#undef ROW_
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}

}  // namespace

extern "C" int tad_distill_loss(int64_t rows, int64_t V, int K, const void* logits, int dtype, int64_t ld, const int64_t* index, const float* value,
                                int64_t ld_t, float tau, const float* row_weight, float grad_scale, float* loss_rows, void* dlogits, int64_t ldd,
                                tad_stream_t stream) {
  TAD_CHECK(rows >= 0 && rows <= INT_MAX && V >= 1 && V <= INT_MAX && K >= 1 && K <= MAX_K, "tad_distill_loss: bad sizes (at most %d entries a row)", MAX_K);
  TAD_CHECK(dtype == TAD_F32 || dtype == TAD_BF16, "tad_distill_loss: bad element type");
  TAD_CHECK(ld >= V && ld_t >= K && (!dlogits || ldd >= V), "tad_distill_loss: bad leading dimension");
  TAD_CHECK(tau > 0.f && tau < INFINITY, "tad_distill_loss: the temperature has to be positive and finite");
  if (rows == 0) return TAD_OK;
  TAD_CHECK(logits && index && value && loss_rows, "tad_distill_loss: null pointer");
  TAD_CHECK(dlogits != logits || ldd == ld, "tad_distill_loss: a gradient in the logits' place needs their row stride");
  const Args A = {rows, V, ld, ld_t, ldd, K, index, value, row_weight, (float)(1.4426950408889634074 / (double)tau), tau, grad_scale, loss_rows};
  return dtype == TAD_F32 ? launch_distill<float>(A, (const float*)logits, (float*)dlogits, (hipStream_t)stream)
                          : launch_distill<bf16_t>(A, (const bf16_t*)logits, (bf16_t*)dlogits, (hipStream_t)stream);
}
