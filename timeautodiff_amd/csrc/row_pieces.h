// Rows of logits of any length and alignment, read 16 bytes a lane.
#pragma once
#include "common.h"

// A row as 16-byte pieces on the aligned grid: piece i holds the elements VEC i - a + (0 .. VEC - 1), a the row's distance
// from the grid; the first and the last may be partly outside the row (-inf there, not loaded).
template <typename T>
struct RowPieces {
  static constexpr int VEC = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(VEC))) T pack;
  const T* x;
  int64_t V, np;
  int a;
  __device__ RowPieces(const T* x_, int64_t V_) : x(x_), V(V_) {
    a = (int)(((uintptr_t)x_ / sizeof(T)) & (VEC - 1));
    np = (V + a + VEC - 1) / VEC;
  }
  __device__ __forceinline__ int64_t first(int64_t i) const { return i * VEC - a; }
  __device__ __forceinline__ pack raw(int64_t i) const {
    const int64_t j = first(i);
    pack p;
    if (j >= 0 && j + VEC <= V) {
      p = *reinterpret_cast<const pack*>(x + j);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) p[e] = j + e >= 0 && j + e < V ? x[j + e] : (T)-INFINITY;
    }
    return p;
  }
  __device__ __forceinline__ void load(int64_t i, float (&v)[VEC]) const {
    const pack p = raw(i);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)p[e];
  }
};
