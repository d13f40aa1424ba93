// gfx950 shared projection with a low-rank adapter of each request beside it:
//
//   out = act( x W^T + bias + scale_g (x A_g^T) B_g^T ),   g the adapter of the row
//
//   adapter_low_kernel   h = scale_g x A_g^T, a tile of rows of one adapter a workgroup
//   adapter_tile_kernel  the product with W over rows in the plan's order, the
//                        h B_g^T of the tile's adapters added to its sums
//   adapter_add_kernel   fp32: h B_g^T added to a projection that is there
//
// Rows are taken in the order of an adapter plan (equal adapters side by side), so 16
// rows of a matrix instruction have few adapters: with streams of 2 frames in their
// own order it would be up to 8.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pk_common.h"
#include "pk_device.h"
#include "pk_tile.h"

namespace pk {

// One step of 16-byte operand chunks: 4 lane groups of 16 bytes a row, 32 columns of
// 16-bit types, 16 of fp32 (four instructions of 4 columns: element e of every
// lane's chunk, the same columns in both operands).
template <typename ST>
struct MmaA {
  static constexpr int COLS = 32;
  __device__ static inline f32x4_t step(u32x4 a, u32x4 b, f32x4_t c) { return MmaL<ST>::k32(a, b, c); }
};
template <>
struct MmaA<float> {
  static constexpr int COLS = 16;
  __device__ static inline f32x4_t step(u32x4 a, u32x4 b, f32x4_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
};

// h is kept as two storage-type parts, high + (h - high), so that the rounding of h
// is 2^-16 (bf16) or 2^-22 (fp16) of it and not 2^-8 or 2^-11 (an h past fp16's range is
// infinite, as it is where x A^T is a product of its own): a row of h is [high
// 0..r-1 | low 0..r-1], r / 4 chunks of 16 bytes, chunk q multiplied with chunk
// q mod r/8 of a row of B.  For ranks up to 16 both parts are one matrix instruction.
// fp32: one part, r / 4 chunks.
template <typename ST>
__device__ static inline int b_chunk(int q, int r) {
  if constexpr (sizeof(ST) == 4) return q;
  const int half = r >> 3;
  return q >= half ? q - half : q;
}

template <typename ST>
struct AdK {
  const ST* x;  // [M][K], stride x_s
  int64_t x_s;
  const ST* w;  // [N][K], stride w_s
  int64_t w_s;
  const ST* bias;  // [N] or nullptr
  const ST* a;     // [G][r][K]
  const ST* b;     // [G][N][r]
  const float* scale;    // [G]
  const int32_t* order;  // [M] plan: row at a position
  const int32_t* ids;    // [M] adapter at a position, -1: none
  const int4* tiles;     // {adapter, first position, rows, 0}
  ST* h;                 // [M][2 r] (fp32: [M][r]) by position
  ST* out;               // [M][N], stride out_s
  int64_t out_s;
  int32_t M, N, K, r, G;
  int32_t mtiles, xm;
};

// row at a position of the plan (positions past the last row, and entries that are no
// row of the batch, give the last row)
template <typename ST>
__device__ static inline int plan_row(const AdK<ST>& p, int pos) {
  return (int)min((uint32_t)p.order[min(pos, p.M - 1)], (uint32_t)p.M - 1u);
}

constexpr int kLowWaves = 8;
constexpr int kLowRows = 32;  // rows of a plan's tile

// h of a tile: the waves split K, 16 RT ranks a workgroup.  Operands come straight from
// memory (every byte is used once a workgroup).
template <typename ST, int RT>
__global__ void __launch_bounds__(64 * kLowWaves) adapter_low_kernel(const AdK<ST> p) {
#pragma clang fp contract(off)
  constexpr int V = Tr<ST>::VEC;
  constexpr int COLS = MmaA<ST>::COLS;
  __shared__ f32x4_t red[kLowWaves * RT * 2 * 64];
  static_assert(2 * RT <= kLowWaves, "a wave finishes at most one sum");
  const int4 tile = p.tiles[blockIdx.x];
  if ((uint32_t)tile.x >= (uint32_t)p.G) return;  // past the last tile
  if (tile.y < 0 || tile.z <= 0 || tile.z > kLowRows || tile.y > p.M - tile.z) return;  // not a plan's
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, kg = lane >> 4;
  const int r0 = blockIdx.y * RT * 16;
  const bool two = tile.z > 16;
  const ST* xp[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) xp[m] = p.x + (int64_t)plan_row(p, tile.y + min(m * 16 + l16, tile.z - 1)) * p.x_s + kg * V;
  const ST* ap[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) ap[j] = p.a + ((int64_t)tile.x * p.r + min(r0 + j * 16 + l16, p.r - 1)) * p.K + kg * V;
  f32x4_t acc[RT][2];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j][0] = acc[j][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int k = wave * COLS; k < p.K; k += kLowWaves * COLS) {
    u32x4 af[RT], xf[2];
    xf[0] = ld16(xp[0] + k);
    if (two) xf[1] = ld16(xp[1] + k);
#pragma unroll
    for (int j = 0; j < RT; ++j) af[j] = ld16(ap[j] + k);
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      acc[j][0] = MmaA<ST>::step(af[j], xf[0], acc[j][0]);
      if (two) acc[j][1] = MmaA<ST>::step(af[j], xf[1], acc[j][1]);
    }
  }
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int m = 0; m < 2; ++m) red[((wave * RT + j) * 2 + m) * 64 + lane] = acc[j][m];
  __syncthreads();
  if (wave >= 2 * RT) return;
  const int row = (wave & 1) * 16 + l16, c = r0 + (wave >> 1) * 16 + kg * 4;
  f32x4_t v = red[wave * 64 + lane];
#pragma unroll
  for (int w = 1; w < kLowWaves; ++w) v += red[(w * RT * 2 + wave) * 64 + lane];
  if (row >= tile.z || c >= p.r) return;  // r is a multiple of 8, c of 4
  const float sc = p.scale[tile.x];
  float f[4] = {v.x * sc, v.y * sc, v.z * sc, v.w * sc};
  if constexpr (sizeof(ST) == 4) {
    st16(p.h + (int64_t)(tile.y + row) * p.r + c, Tr<float>::pack(f));
  } else {
    float lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float hi = round_to<ST>(f[e]);
      lo[e] = fabsf(hi) < __builtin_inff() ? f[e] - hi : 0.f;
    }
    ST* const q = p.h + (int64_t)(tile.y + row) * 2 * p.r + c;
    *reinterpret_cast<u32x2*>(q) = pack4<ST>(f);
    *reinterpret_cast<u32x2*>(q + p.r) = pack4<ST>(lo);
  }
}

// acc[m][n] += h B^T for TM x TN products of rows pos0 + 16 m and columns c0 + 16 n, one
// pass for each adapter among the rows; of the adapters, part `wk` of WK.  Columns of a
// product (the rows of the batch) are independent, so where only some of 16 rows have
// the adapter the product is taken for all of them and kept for those: what a row gets
// depends on its own adapter alone, an infinity or NaN in another's B does not reach it.
template <typename ST, int TM, int TN, int WK>
__device__ static inline void add_low(const AdK<ST>& p, const int (&id)[TM], int pos0, int c0, int wk, int lane,
                                      f32x4_t (&acc)[TM][TN]) {
  constexpr int V = Tr<ST>::VEC;
  const int l16 = lane & 15, kg = lane >> 4;
  const int chunks = p.r >> 2, hs = sizeof(ST) == 4 ? p.r : 2 * p.r;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  const ST* hp[TM];
  uint64_t left[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    left[m] = __ballot(id[m] >= 0);
    hp[m] = p.h + (int64_t)min(pos0 + m * 16 + l16, p.M - 1) * hs;
  }
  for (int turn = 0;; turn = turn == WK - 1 ? 0 : turn + 1) {
    int g = -1;
#pragma unroll
    for (int m = TM - 1; m >= 0; --m)
      if (left[m]) g = __builtin_amdgcn_readlane(id[m], __builtin_ctzll(left[m]));
    if (g < 0) break;
    uint64_t has[TM];
    bool whole = false;
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      has[m] = __ballot(id[m] == g);
      left[m] &= ~has[m];
      whole |= has[m] == ~(uint64_t)0;
    }
    if (WK > 1 && turn != wk) continue;
    const ST* const bp = p.b + ((int64_t)g * p.N + c0 + l16) * p.r;
    auto b_of = [&](int n, int q) { return q < chunks ? ld16(bp + (int64_t)n * 16 * p.r + b_chunk<ST>(q, p.r) * V) : zero; };
    if (whole) {
      for (int q = kg; q - kg < chunks; q += 4) {
        u32x4 bf[TN];
#pragma unroll
        for (int n = 0; n < TN; ++n) bf[n] = b_of(n, q);
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          if (has[m] != ~(uint64_t)0) continue;
          const u32x4 hf = q < chunks ? ld16(hp[m] + q * V) : zero;
#pragma unroll
          for (int n = 0; n < TN; ++n) acc[m][n] = MmaA<ST>::step(bf[n], hf, acc[m][n]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      if (has[m] == 0 || has[m] == ~(uint64_t)0) continue;
      f32x4_t d[TN];
#pragma unroll
      for (int n = 0; n < TN; ++n) d[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int q = kg; q - kg < chunks; q += 4) {
        const u32x4 hf = q < chunks ? ld16(hp[m] + q * V) : zero;
#pragma unroll
        for (int n = 0; n < TN; ++n) d[n] = MmaA<ST>::step(b_of(n, q), hf, d[n]);
      }
      if (id[m] == g) {
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] += d[n];
      }
    }
  }
}

template <int SILU>
__device__ static inline float ad_act(float v) {
  if constexpr (SILU) return v / (1.f + __expf(-v));
  return v;
}

// The product with W: BM x BN outputs a workgroup, both operands staged in LDS as in
// lin_tile_kernel, the rows of x and of the output those that the plan's order names.
// The adapters' part is summed first, while the first stages are on their way.
template <typename ST, int BM, int BN, int WM, int WN, int WK, int BK, int S, int SILU>
__global__ void __launch_bounds__(64 * WM * WN * WK) adapter_tile_kernel(const AdK<ST> p) {
#pragma clang fp contract(off)
  constexpr int NW = WM * WN * WK;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int CH = BK / 8;
  constexpr int kStage = (BM + BN) * BK * 2;
  constexpr int LPS = kStage / 1024 / NW;
  static_assert(BK % 64 == 0, "the permutation stays within a row's stage: whole groups of 8 chunks");
  static_assert(kStage % (1024 * NW) == 0 && (BM * CH) % 64 == 0, "whole waves of chunks");
  constexpr int KS = BK / 32 / WK;
  constexpr int OS = BN + 8;
  constexpr int kOut = BM * OS * 2;
  constexpr int kRed = WK > 1 ? (WK - 1) * BM * BN * 4 : 0;
  constexpr int kSmem = S * kStage > kOut + kRed ? S * kStage : kOut + kRed;
  __shared__ __align__(16) unsigned char smem[kSmem];
  __shared__ int32_t ord[BM];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, kg = lane >> 4;
  const int wk = wave / (WM * WN), wm = (wave / WN) % WM, wn = wave % WN;
  int mt_i, nt_i;
  xcd_tile(p.mtiles, p.xm, mt_i, nt_i);
  const int row0 = mt_i * BM, n0 = nt_i * BN;

  // positions past the last row read the last row and store nothing
  for (int i = threadIdx.x; i < BM; i += 64 * NW) ord[i] = plan_row(p, row0 + i);
  int id[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int pos = row0 + (wm * TM + m) * 16 + l16;
    id[m] = pos < p.M ? p.ids[pos] : -1;
    if ((uint32_t)id[m] >= (uint32_t)p.G) id[m] = -1;
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t rx = bytes_rsrc(p.x, (uint32_t)((p.M - 1) * p.x_s + p.K) * 2u);
  const __amdgpu_buffer_rsrc_t rw = bytes_rsrc(p.w, (uint32_t)((p.N - 1) * p.w_s + p.K) * 2u);
  uint32_t off[LPS];
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const int c = (i * NW + wave) * 64 + lane;
    const int r = c / CH, pos = c % CH;
    const int ch = (pos & ~7) | ((pos ^ r) & 7);
    off[i] = r < BM ? (uint32_t)(ord[r] * p.x_s + ch * 8) * 2u : (uint32_t)((n0 + r - BM) * p.w_s + ch * 8) * 2u;
  }
  auto issue = [&](int st, int k) {
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const int base = (i * NW + wave) * 64;
      load_lds16(base < BM * CH ? rx : rw, smem + st * kStage + base * 16, off[i], k * 2);
    }
  };
  f32x4_t acc[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int iters = p.K / BK;
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < iters) issue(s, s * BK);
  add_low<ST, TM, TN, WK>(p, id, row0 + wm * TM * 16, n0 + wn * TN * 16, wk, lane, acc);
  int st = 0;
  for (int it = 0; it < iters; ++it) {
    if (it + S - 2 < iters)
      wait_vm<(S - 2) * LPS>();
    else
      wait_vm<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (it + S - 1 < iters) issue(st == 0 ? S - 1 : st - 1, (it + S - 1) * BK);
    const unsigned char* xs = smem + st * kStage;
    const unsigned char* ws = xs + BM * BK * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ch = (wk * KS + s) * 4 + kg;
      u32x4 xf[TM], wf[TN];
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const int r = (wm * TM + m) * 16 + l16;
        xf[m] = *reinterpret_cast<const u32x4*>(xs + r * BK * 2 + ((ch & ~7) | ((ch ^ r) & 7)) * 16);
      }
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        const int r = (wn * TN + n) * 16 + l16;
        wf[n] = *reinterpret_cast<const u32x4*>(ws + r * BK * 2 + ((ch & ~7) | ((ch ^ r) & 7)) * 16);
      }
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = MmaL<ST>::k32(wf[n], xf[m], acc[m][n]);
    }
    st = st == S - 1 ? 0 : st + 1;
  }
  __syncthreads();
  sum_parts<BM, BN, WM * WN, WK>(smem, kOut, acc, wave, lane);
  ST* const os = reinterpret_cast<ST*>(smem);
  if (wk == 0) {
#pragma unroll
    for (int n = 0; n < TN; ++n) {
      const int c = (wn * TN + n) * 16 + kg * 4;
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = from_st(p.bias[n0 + c + e]);
      }
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        float f[4] = {acc[m][n].x, acc[m][n].y, acc[m][n].z, acc[m][n].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = ad_act<SILU>(f[e] + b[e]);
        *reinterpret_cast<u32x2*>(os + ((wm * TM + m) * 16 + l16) * OS + c) = pack4<ST>(f);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BM * BN / 8; i += 64 * NW) {
    const int r = i / (BN / 8), c = (i % (BN / 8)) * 8;
    if (row0 + r < p.M) st16(p.out + (int64_t)ord[r] * p.out_s + n0 + c, *reinterpret_cast<const u32x4*>(os + r * OS + c));
  }
}

// fp32: out = act(out + h B^T), 16 rows x 64 columns a wave, out read in the layout of
// the matrix instruction's sums (4 columns of a row a lane).
template <int SILU>
__global__ void __launch_bounds__(256) adapter_add_kernel(const AdK<float> p) {
  constexpr int TN = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, kg = lane >> 4;
  const int pos = blockIdx.x * 16 + l16, c0 = (blockIdx.y * 4 + wave) * TN * 16;
  if (c0 >= p.N) return;  // the whole wave; no barrier below
  int id[1] = {pos < p.M ? p.ids[pos] : -1};
  if ((uint32_t)id[0] >= (uint32_t)p.G) id[0] = -1;
  float* const q = p.out + (int64_t)plan_row(p, pos) * p.out_s + c0 + kg * 4;
  f32x4_t acc[1][TN];
#pragma unroll
  for (int n = 0; n < TN; ++n) acc[0][n] = __builtin_bit_cast(f32x4_t, ld16(q + n * 16));
  add_low<float, 1, TN, 1>(p, id, blockIdx.x * 16, c0, 0, lane, acc);
  if (pos >= p.M) return;
#pragma unroll
  for (int n = 0; n < TN; ++n) {
    f32x4_t v = acc[0][n];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ad_act<SILU>(v[e]);
    st16(q + n * 16, __builtin_bit_cast(u32x4, v));
  }
}

namespace {

template <typename ST>
int launch_low(const AdK<ST>& k, int max_tiles, hipStream_t s) {
  const int rt = (k.r + 15) / 16, per = rt < 4 ? rt : 4;
  const dim3 grid((unsigned)max_tiles, (unsigned)((rt + per - 1) / per)), block(64 * kLowWaves);
  switch (per) {
    case 1: hipLaunchKernelGGL((adapter_low_kernel<ST, 1>), grid, block, 0, s, k); break;
    case 2: hipLaunchKernelGGL((adapter_low_kernel<ST, 2>), grid, block, 0, s, k); break;
    case 3: hipLaunchKernelGGL((adapter_low_kernel<ST, 3>), grid, block, 0, s, k); break;
    default: hipLaunchKernelGGL((adapter_low_kernel<ST, 4>), grid, block, 0, s, k); break;
  }
  return check_launch("pk_adapter_linear");
}

template <typename ST, int BM, int BN, int WM, int WN, int WK, int BK, int S, int SILU>
int launch_tile(AdK<ST> k, hipStream_t s) {
  k.mtiles = (k.M + BM - 1) / BM;
  const int nt = k.N / BN;
  k.xm = xcd_split(k.mtiles, nt, BM, BN);
  dim3 grid((unsigned)(k.mtiles * nt));
  if (k.xm > 0 && k.mtiles / k.xm <= 65535 && nt / (8 / k.xm) <= 65535)
    grid = dim3(8u, (unsigned)(k.mtiles / k.xm), (unsigned)(nt / (8 / k.xm)));
  else
    k.xm = 0;
  hipLaunchKernelGGL((adapter_tile_kernel<ST, BM, BN, WM, WN, WK, BK, S, SILU>), grid, dim3(64 * WM * WN * WK), 0, s, k);
  return check_launch("pk_adapter_linear");
}

template <typename ST, int SILU>
int launch_product(const AdK<ST>& k, hipStream_t s) {
  return launch_tile<ST, 64, 64, 2, 2, 2, 64, 4, SILU>(k, s);
}

bool rows_ok(int64_t rows, int64_t stride, int64_t width, int vec) {
  return stride >= 0 && stride % vec == 0 && (rows <= 1 || stride >= width) && (rows - 1) * stride + width < (int64_t{1} << 31);
}

template <typename ST>
int adapter_typed(const pk_adapter_linear_args* a, hipStream_t s) {
  const char* what = "pk_adapter_linear";
  constexpr bool kF32 = sizeof(ST) == 4;
  if (a->rows < 0) return fail(PK_ERR_INVALID, "%s: rows %d < 0", what, a->rows);
  if (a->n <= 0 || a->n % 64 != 0 || a->k <= 0 || a->k % 64 != 0)
    return fail(PK_ERR_UNSUPPORTED, "%s: n %d and k %d must be multiples of 64", what, a->n, a->k);
  if (a->rank <= 0 || a->rank % 8 != 0 || a->rank > PK_ADAPTER_MAX_RANK)
    return fail(PK_ERR_UNSUPPORTED, "%s: rank %d must be a multiple of 8, at most %d", what, a->rank, PK_ADAPTER_MAX_RANK);
  if (a->num_adapters <= 0 || a->num_adapters > PK_ADAPTER_MAX)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d adapters (built: 1 to %d)", what, a->num_adapters, PK_ADAPTER_MAX);
  if (a->activation != PK_ACT_NONE && a->activation != PK_ACT_SILU)
    return fail(PK_ERR_INVALID, "%s: activation %d must be none or SiLU", what, a->activation);
  if (a->max_tiles < 0) return fail(PK_ERR_INVALID, "%s: max_tiles %d < 0", what, a->max_tiles);
  if (a->rows == 0) return PK_OK;
  if (kF32 && (a->weight || a->bias))
    return fail(PK_ERR_INVALID, "%s: fp32 adds to a projection that out holds; weight and bias must be NULL", what);
  const void* ptrs[9] = {a->x,     a->a,  a->b,         kF32 ? a->x : a->weight, a->bias ? a->bias : a->x,
                         a->tiles, a->out, a->workspace, a->scale};
  for (const void* q : ptrs) {
    if (!q) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
    if (q != a->scale && !aligned16(q)) return fail(PK_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  }
  if (!a->order || !a->ids) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  constexpr int V = Tr<ST>::VEC;
  if (!rows_ok(a->rows, a->x_stride, a->k, V) || (!kF32 && !rows_ok(a->n, a->weight_stride, a->k, V)) ||
      !rows_ok(a->rows, a->out_stride, a->n, V))
    return fail(PK_ERR_INVALID, "%s: row strides must be multiples of %d elements, at least the row, and a tensor below 2^31 elements",
                what, V);
  AdK<ST> k{};
  k.x = static_cast<const ST*>(a->x);
  k.x_s = a->x_stride;
  k.w = static_cast<const ST*>(a->weight);
  k.w_s = a->weight_stride;
  k.bias = static_cast<const ST*>(a->bias);
  k.a = static_cast<const ST*>(a->a);
  k.b = static_cast<const ST*>(a->b);
  k.scale = a->scale;
  k.order = a->order;
  k.ids = a->ids;
  k.tiles = reinterpret_cast<const int4*>(a->tiles);
  k.h = static_cast<ST*>(a->workspace);
  k.out = static_cast<ST*>(a->out);
  k.out_s = a->out_stride;
  k.M = a->rows;
  k.N = a->n;
  k.K = a->k;
  k.r = a->rank;
  k.G = a->num_adapters;
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  if (a->max_tiles > 0) {
    const int rc = launch_low(k, a->max_tiles, s);
    if (rc != PK_OK) return rc;
  }
  const bool silu = a->activation == PK_ACT_SILU;
  if constexpr (kF32) {
    const dim3 grid((unsigned)((k.M + 15) / 16), (unsigned)((k.N + 255) / 256));
    if (silu)
      hipLaunchKernelGGL(adapter_add_kernel<1>, grid, dim3(256), 0, s, k);
    else
      hipLaunchKernelGGL(adapter_add_kernel<0>, grid, dim3(256), 0, s, k);
    return check_launch(what);
  } else {
    return silu ? launch_product<ST, 1>(k, s) : launch_product<ST, 0>(k, s);
  }
}

}  // namespace
}  // namespace pk

extern "C" int64_t pk_adapter_workspace_bytes(int32_t rows, int32_t rank) {
  return rows > 0 && rank > 0 ? (int64_t)rows * rank * 4 : 0;
}

extern "C" int pk_adapter_linear(const pk_adapter_linear_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_adapter_linear: args is NULL");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (args->dtype) {
    case PK_DTYPE_F32: return pk::adapter_typed<float>(args, s);
    case PK_DTYPE_F16: return pk::adapter_typed<_Float16>(args, s);
    case PK_DTYPE_BF16: return pk::adapter_typed<pk::bf16_t>(args, s);
    default: return pk::fail(PK_ERR_INVALID, "pk_adapter_linear: unknown dtype %d", args->dtype);
  }
}
