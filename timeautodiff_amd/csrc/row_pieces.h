// Rows of logits of any length and alignment, read 16 bytes a lane.
#pragma once
#include "common.h"

// A row of at least VEC elements as pieces of 16 bytes, VEC elements from its first on, wherever that lies (vector loads need
// the alignment of an element only).  Where VEC does not divide the row, the last piece is moved back to end with it;
// load() gives what the piece before it holds already as -inf.
template <typename T>
struct RowPieces {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T pack __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
  const T* x;
  int64_t V, np;
  __device__ RowPieces(const T* x_, int64_t V_) : x(x_), V(V_), np((V_ + VEC - 1) / VEC) {}
  __device__ __forceinline__ int64_t first(int64_t i) const { return i * VEC + VEC <= V ? i * VEC : V - VEC; }
  __device__ __forceinline__ void load(int64_t i, float (&v)[VEC]) const {
    const int64_t j = first(i);
    const int again = (int)(i * VEC - j);
    const pack p = *reinterpret_cast<const pack*>(x + j);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)p[e];
    if (again) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = e < again ? -INFINITY : v[e];
    }
  }
};
