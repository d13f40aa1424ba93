// Pieces of the gfx950 matrix-product kernels: matrix-core operands, loads straight
// to LDS and their waits, the tile order over the XCDs, sums over the parts of K.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pk_device.h"

namespace pk {

template <typename ST>
struct MmaL;
template <>
struct MmaL<_Float16> {
  typedef _Float16 H8 __attribute__((ext_vector_type(8)));
  __device__ static inline f32x4_t k32(u32x4 a, u32x4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  }
};
template <>
struct MmaL<bf16_t> {
  typedef __bf16 H8 __attribute__((ext_vector_type(8)));
  __device__ static inline f32x4_t k32(u32x4 a, u32x4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  }
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename ST>
__device__ static inline u32x2 pack4(const float* f) {
  u32x2 v;
  if constexpr (sizeof(ST) == 2 && __is_same(ST, bf16_t)) {
    v.x = bf16_pair_bits(f[0], f[1]);
    v.y = bf16_pair_bits(f[2], f[3]);
  } else {
    v.x = Tr<_Float16>::two(f);
    v.y = Tr<_Float16>::two(f + 2);
  }
  return v;
}

// Tile (m, n) of a workgroup: workgroups go to the XCDs in turn in launch order.
// xm > 0: grid (8, row tiles, column tiles of an XCD): the XCDs take an xm x 8/xm
// grid of equal blocks of tiles (the host picks xm, a power of two, so that a
// block's rows and weight columns together are fewest: what each XCD's L2
// fetches).  xm == 0 (the tiles do not divide): grid (tiles), contiguous runs of
// them an XCD, rows fastest.
__device__ static inline void xcd_tile(int mtiles, int xm, int& m, int& n) {
  if (xm > 0) {
    const int x = blockIdx.x, lg = xm == 1 ? 0 : xm == 2 ? 1 : xm == 4 ? 2 : 3;
    m = (x & (xm - 1)) * gridDim.y + blockIdx.y;
    n = (x >> lg) * gridDim.z + blockIdx.z;
    return;
  }
  const int total = gridDim.x, x = blockIdx.x & 7, j = blockIdx.x >> 3;
  const int t = x * (total >> 3) + min(x, total & 7) + j;
  m = t % mtiles;
  n = t / mtiles;
}

// `bytes` readable from base; a read past them gives zeros
__device__ static inline __amdgpu_buffer_rsrc_t bytes_rsrc(const void* base, uint32_t bytes) {
  // word 3 0x00020000: 32-bit data format, the setting untyped loads need on CDNA
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

// 16 bytes a lane to lds + 16 lane (lds wave-uniform)
__device__ static inline void load_lds16(const __amdgpu_buffer_rsrc_t r, unsigned char* lds, uint32_t off, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, soff, 0, 0);
}

// vmcnt(n): at most n of the wave's memory reads still in flight
template <int N>
__device__ static inline void wait_vm() {
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N & 0x30) << 10));
}

// The sums of the WK parts of K meet in LDS (at smem + at); waves are numbered
// (wk WM + wm) WN + wn, the waves wk == 0 end with the sums.
template <int BM, int BN, int WMN, int WK, int TM, int TN>
__device__ static inline void sum_parts(unsigned char* smem, int at, f32x4_t (&acc)[TM][TN], int wave, int lane) {
  if constexpr (WK > 1) {
    f32x4_t* const red = reinterpret_cast<f32x4_t*>(smem + at);
    if (wave >= WMN) {
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) red[((wave - WMN) * TM * TN + m * TN + n) * 64 + lane] = acc[m][n];
    }
    __syncthreads();
    if (wave < WMN) {
#pragma unroll
      for (int w = 1; w < WK; ++w)
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
          for (int n = 0; n < TN; ++n) acc[m][n] += red[((wave + (w - 1) * WMN) * TM * TN + m * TN + n) * 64 + lane];
    }
  }
}

// the split of the XCDs over rows (see xcd_tile)
inline int xcd_split(int mtiles, int ntiles, int bm, int bn) {
  int best = 0;
  int64_t cost = 0;
  for (int xm = 1; xm <= 8; xm *= 2) {
    if (mtiles % xm != 0 || ntiles % (8 / xm) != 0) continue;
    const int64_t c = (int64_t)(mtiles / xm) * bm + (int64_t)(ntiles / (8 / xm)) * bn;
    if (best == 0 || c < cost) {
      best = xm;
      cost = c;
    }
  }
  return best;
}

}  // namespace pk
