// Distillation loss of a student's logits against a teacher's top logits, and its gradient (gfx950).
//
//   q_k = softmax over the row's valid entries of value[r, k] / tau        (an index outside [0, V) is no entry)
//   p_j = softmax over the row of logits[r, j] / tau
//   loss[r] = w_r tau^2 sum_k q_k (ln q_k - ln p[index_k]),   dlogits[r, j] = grad_scale w_r tau (p_j - sum of the q_k with index_k = j)
//
// Statistics and sums in fp32.  The logits are read and the gradient written once each: HBM bounds it.
#include <limits.h>
#include <math.h>

#include "common.h"

namespace {

constexpr int MAX_K = 1024;
constexpr float LOWEST = -3.4028234663852886e38f;

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
__device__ __forceinline__ float wave_max(float v) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
template <int NW>
__device__ __forceinline__ float block_max(float v, float* s) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = s[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) t = fmaxf(t, s[w]);
  return t;
}

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(256) void distill_row_kernel(int64_t rows, int64_t V, int K, const T* logits, int64_t ld,
                                                          const int64_t* __restrict__ index, const float* __restrict__ value, int64_t ld_t,
                                                          float tau, const float* __restrict__ weight, float grad_scale, float* __restrict__ loss,
                                                          T* dlogits, int64_t ldd) {
  __shared__ float red[4];
  __shared__ float q[MAX_K];
  __shared__ int64_t at[MAX_K];
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const T* x = logits + r * ld;
  const float w = weight ? weight[r] : 1.f;
  const float it = 1.f / tau;
  float m = LOWEST;
  if (w != 0.f)
    for (int64_t j = tid; j < V; j += 256) m = fmaxf(m, (float)x[j]);
  m = block_max<4>(m, red);
  float z = 0.f;
  if (w != 0.f)
    for (int64_t j = tid; j < V; j += 256) z += expf(((float)x[j] - m) * it);
  z = block_sum<4>(z, red);
  if (w == 0.f || z == 0.f) {          // the row counts nothing, or no student logit is finite
    if (tid == 0) loss[r] = 0.f;
    if (dlogits)
      for (int64_t j = tid; j < V; j += 256) dlogits[r * ldd + j] = (T)0.f;
    return;
  }
  const float lnz = logf(z);
  float tm = LOWEST;
  for (int k = tid; k < K; k += 256) {
    const int64_t i = index[r * ld_t + k];
    at[k] = (uint64_t)i < (uint64_t)V ? i : -1;
    if (at[k] >= 0) tm = fmaxf(tm, value[r * ld_t + k]);
  }
  tm = block_max<4>(tm, red);
  float tz = 0.f;
  for (int k = tid; k < K; k += 256) {
    q[k] = at[k] >= 0 ? expf((value[r * ld_t + k] - tm) * it) : 0.f;
    tz += q[k];
  }
  tz = block_sum<4>(tz, red);
  const float lntz = tz > 0.f ? logf(tz) : 0.f, itz = tz > 0.f ? 1.f / tz : 0.f;
  float l = 0.f;
  for (int k = tid; k < K; k += 256) {
    q[k] *= itz;
    if (q[k] > 0.f) l += q[k] * (((value[r * ld_t + k] - tm) * it - lntz) - (((float)x[at[k]] - m) * it - lnz));
  }
  l = block_sum<4>(l, red);
  if (tid == 0) loss[r] = w * tau * tau * l;
  if (!dlogits) return;
  const float iz = tz > 0.f ? 1.f / z : 0.f, g = grad_scale * w * tau;
  T* d = dlogits + r * ldd;
  float mine[MAX_K / 256];             // the student's p at this thread's entries, before the row may be overwritten
  for (int k = tid, n = 0; k < K; k += 256, ++n) mine[n] = at[k] >= 0 ? expf(((float)x[at[k]] - m) * it) * iz : 0.f;
  __syncthreads();
  for (int64_t j = tid; j < V; j += 256) d[j] = (T)(g * (expf(((float)x[j] - m) * it) * iz));
  __syncthreads();
  for (int k = tid, n = 0; k < K; k += 256, ++n) {
    if (at[k] < 0) continue;
    float s = 0.f;
    bool first = true;
    for (int o = 0; o < K; ++o) {
      if (at[o] != at[k]) continue;
      if (o < k) first = false;
      s += q[o];
    }
    if (first) d[at[k]] = (T)(g * (mine[n] - s));
  }
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
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TAD_F32)
    hipLaunchKernelGGL(distill_row_kernel<float>, dim3((unsigned)rows), dim3(256), 0, s, rows, V, K, (const float*)logits, ld, index, value, ld_t, tau,
                       row_weight, grad_scale, loss_rows, (float*)dlogits, ldd);
  else
    hipLaunchKernelGGL(distill_row_kernel<bf16_t>, dim3((unsigned)rows), dim3(256), 0, s, rows, V, K, (const bf16_t*)logits, ld, index, value, ld_t,
                       tau, row_weight, grad_scale, loss_rows, (bf16_t*)dlogits, ldd);
  TAD_LAUNCH_CHECK();
  return TAD_OK;
}
