// Reductions and scans over groups of lanes of a wave: moves inside rows of 16 lanes by DPP, rows by scalar lane reads.
#pragma once
#include "common.h"

typedef unsigned long long u64;

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

// LDS accesses of a wave before and after this are in order for its own lanes (the hardware keeps a wave's LDS order; this keeps
// the compiler to it)
__device__ __forceinline__ void lds_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
