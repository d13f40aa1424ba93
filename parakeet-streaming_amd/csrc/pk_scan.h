// Sums over the lanes of a wave and the waves of a workgroup, in order, and host-side
// arithmetic of page sizes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pk {

// inclusive sum over the 64 lanes of a wave
template <typename T>
__device__ static inline T wave_scan(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  return v;
}

// exclusive sum over a workgroup of NW waves; `sum`: of all
template <int NW, typename T>
__device__ static inline T block_scan(T v, T* lds, T& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T inc = wave_scan(v);
  if (lane == 63) lds[wave] = inc;
  __syncthreads();
  T before = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const T x = lds[w];
    if (w < wave) before += x;
    sum += x;
  }
  __syncthreads();
  return before + inc - v;
}

// s with x == 2^s, -1 where there is none
inline int log2_of(int32_t x) {
  for (int s = 0; s < 31; ++s)
    if ((int32_t{1} << s) == x) return s;
  return -1;
}

}  // namespace pk
