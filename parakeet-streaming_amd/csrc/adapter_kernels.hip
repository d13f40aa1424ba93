// gfx950 shared projection with a low-rank adapter of each request beside it:
//
//   out = act( x W^T + bias + scale_g (x A_g^T) B_g^T ),   g the adapter of the row
//
//   adapter_low_kernel   h = scale_g x A_g^T, a tile of rows of one adapter a workgroup
//   adapter_tile_kernel  the product with W over rows in the plan's order, the
//                        h B_g^T of the tile's adapters added to its sums
//   adapter_few_kernel   both in one launch, for few rows with few adapters among them
//
// Rows are taken in the order of an adapter plan (equal adapters side by side), so 16
// rows of a matrix instruction have few adapters: with streams of 2 frames in their
// own order it would be up to 8.

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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
// is 2^-16 (bf16, from 2^-110 up) or 2^-22 (fp16) of it and not 2^-8 or 2^-11: a row of h is [high
// 0..r-1 | low 0..r-1], r / 4 chunks of 16 bytes, chunk q multiplied with chunk
// q mod r/8 of a row of B.  For ranks up to 16 both parts are one matrix instruction.
// fp32: one part, r / 4 chunks.  Where K is split over workgroups (parts > 1) a row of h
// is the parts' rows one after another: their sum is taken by the product with B.
//
// fp16 holds 2^-24 to 65504 where h is any fp32 number, so its rows are kept in units of a
// power of two (row_unit) that the sums are multiplied with once h B^T is taken.  A workgroup
// of adapter_low_kernel knows its part of K and its 64 ranks only: each such piece of a row
// has its own unit, and the product with B brings them to the row's largest (to_unit).  What
// is below fp16's smallest step then is below 2^-36 of the row's largest entry.  The units, 4
// floats, are a row's end, in lines that h's readers load anyway.  They cost 0.2 - 0.7 us of a
// call (840 rows 4096 -> 1024, r 32: 26.9 us with, 26.5 without; 4000 rows 512 -> 2048 SiLU: 23.7
// and 22.6), 4 where a row of 128 ranks has two pieces (3584 rows 1024 -> 4096: 66 and 62).
constexpr int kLowChunks = 16, kLowRow = kLowChunks * 16;  // chunks and bytes of a row of h in LDS

template <typename ST>
__device__ static inline int b_chunk(int q, int r) {
  return (int)((uint32_t)q % (uint32_t)(sizeof(ST) == 4 ? r >> 2 : r >> 3));
}

// How the product takes a row of h: `copies` of `width` chunks each multiplied with the same
// chunks of B, `block` chunks of every copy a turn, 4 of them a step.  Staged rows (LDS)
// read B once for the high and low parts of h and of each part of K (256 adapters of rank
// 64: 3584 rows 1024 -> 4096 81 us so and 94 with a read each, 840 rows 60 and 78), except
// ranks below 32, where a step of 4 chunks would be half empty; rows from memory take
// one chunk after another.
struct LowOrder {
  int copies, width, block;
  int shift;  // of a block, staged: a power of two
};
template <typename ST, bool LDS>
__device__ static inline LowOrder low_order(int r, int parts) {
  const int copies = !LDS ? 1 : sizeof(ST) == 4 ? parts : r >= 32 ? 2 * parts : 1;
  const int width = (r >> 2) * parts / copies;
  return LowOrder{copies, width, LDS ? kLowChunks / copies : width, 4 - (copies >> 1)};
}

template <typename ST>
constexpr bool kUnits = __is_same(ST, _Float16);
constexpr int kMaxUnits = 4;  // pieces of a row of h: 2 parts of K, 64 of 128 ranks

// bytes of a row of h
template <typename ST>
__host__ __device__ constexpr uint32_t low_row(int r, int parts) {
  return (uint32_t)(r * 4 * parts) + (kUnits<ST> ? 4 * kMaxUnits : 0);
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
  ST* h;                 // [M] rows by position: [parts][2 r], fp16 units behind; fp32 [parts][r]
  ST* out;               // [M][N], stride out_s
  int64_t out_s;
  int32_t M, N, K, r, G;
  int32_t parts, kpart;  // parts of K, columns of one (a multiple of 64)
  int32_t mtiles, xm;
  int32_t units;  // pieces of a row of h (fp16)
};

// row at a position of the plan (positions past the last row, and entries that are no
// row of the batch, give the last row)
template <typename ST>
__device__ static inline int plan_row(const AdK<ST>& p, int pos) {
  return (int)min((uint32_t)p.order[min(pos, p.M - 1)], (uint32_t)p.M - 1u);
}

constexpr int kLowWaves = 8;
constexpr int kLowRows = 32;  // rows of a plan's tile

// an offset that no tensor here reaches (each is below 2^31 bytes): such a load gives zeros
constexpr uint32_t kNowhere = 0x80000000u;
__device__ static inline u32x4 load16(const __amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ static inline u32x2 load8(const __amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
}

// 4 fp16 entries in fp32
__device__ static inline u32x4 wide(u32x2 v) {
  float f[4];
  Tr<_Float16>::two(v.x, f);
  Tr<_Float16>::two(v.y, f + 2);
  return Tr<float>::pack(f);
}
__device__ static inline u32x4 wide(u32x4 v) { return v; }

// 4 ranks of a row of h, scaled (and in the row's units), at q (their low parts r elements on)
template <typename ST>
__device__ static inline void store_low(f32x4_t v, float sc, float down, ST* q, int r) {
  float f[4] = {v.x * sc, v.y * sc, v.z * sc, v.w * sc};
  if constexpr (kUnits<ST>) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] *= down;
  }
  if constexpr (sizeof(ST) == 4) {
    st16(q, Tr<float>::pack(f));
  } else {
    float lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float hi = round_to<ST>(f[e]);
      lo[e] = fabsf(hi) < __builtin_inff() ? f[e] - hi : 0.f;
    }
    *reinterpret_cast<u32x2*>(q) = pack4<ST>(f);
    *reinterpret_cast<u32x2*>(q + r) = pack4<ST>(lo);
  }
}

// the largest finite magnitude, scaled, among the ranks that the 4 lanes of a row have
__device__ static inline float largest_of_row(f32x4_t v, float sc) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float f = fabsf(v[e] * sc);
    m = f < __builtin_inff() ? fmaxf(m, f) : m;
  }
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Units of a row whose largest finite magnitude is m: times `down` m is in [2^14, 2^15) (less
// below 2^-112), `up` is its inverse; both are normal powers of two.
struct RowUnit {
  float down, up;
};
__device__ static inline RowUnit row_unit(float m) {
  const uint32_t e = min(max(__float_as_uint(m) >> 23, 15u), 254u);
  return RowUnit{__uint_as_float((268u - e) << 23), __uint_as_float((e - 14u) << 23)};
}

// `own` / `most`, powers of two with own <= most, as the product of two fp16 numbers (at
// least 2^-38: entries that are below that step of a row's largest one)
__device__ static inline uint32_t unit_ratio(float own, float most) {
  const uint32_t d = min((__float_as_uint(most) - __float_as_uint(own)) >> 23, 38u);
  const uint32_t d1 = min(d, 14u), d2 = d - d1;
  return (15u - d1) << 10 | (d2 < 15u ? (15u - d2) << 10 : 1u << (24u - d2)) << 16;
}

// 8 entries of h in the row's units
__device__ static inline u32x4 to_unit(u32x4 h, uint32_t ratio) {
  typedef MmaL<_Float16>::H8 H8;
  const _Float16 a = __builtin_bit_cast(_Float16, (uint16_t)ratio), b = __builtin_bit_cast(_Float16, (uint16_t)(ratio >> 16));
  return __builtin_bit_cast(u32x4, __builtin_bit_cast(H8, h) * (H8)a * (H8)b);
}

// the piece of a row of h that chunk q of copy c is in
__device__ static inline int piece_of(const LowOrder& o, int r, int c, int q) {
  int part = c >> 1;  // copies: high and low of each part of K
  if (o.copies == 1) {
    part = q >= r >> 2 ? 1 : 0;
    q -= part * (r >> 2);
    if (q >= r >> 3) q -= r >> 3;
  }
  return part * ((r + 63) >> 6) + (q >> 3);
}

// h of a tile: its 32 rows of x and 16 RT rows of A through LDS, 512 bytes of each a
// stage, S stages on their way (whole lines; read straight from memory as matrix
// operands, 16 rows of 64 bytes an instruction, a CU moved 16-34 GB/s).  The waves take
// a step of 4 chunks a lane group of each stage and their sums meet at the end.  Columns past
// the part's end are loaded from its start and not multiplied.
template <typename ST, int RT, int S>
__global__ void __launch_bounds__(64 * kLowWaves) adapter_low_kernel(const AdK<ST> p) {
#pragma clang fp contract(off)
  constexpr int E = sizeof(ST), V = 16 / E, COLS = MmaA<ST>::COLS;
  constexpr int CH = 4 * kLowWaves, ROW = CH * 16, BK = ROW / E;  // a wave's step each
  constexpr int NR = kLowRows + 16 * RT, kStage = NR * ROW;
  constexpr int LPS = NR * CH / 64 / kLowWaves;
  static_assert(NR * CH % (64 * kLowWaves) == 0 && BK == COLS * kLowWaves, "whole waves of chunks, a step a wave");
  constexpr int kRed = kLowWaves * RT * 2 * 64 * 16;
  static_assert(S * kStage >= kRed + 2 * RT * 16 * 4, "a row's largest entries beside the sums");
  __shared__ __align__(16) unsigned char smem[S * kStage > kRed ? S * kStage : kRed];
  static_assert(2 * RT <= kLowWaves, "a wave finishes at most one sum");
  const int4 tile = p.tiles[blockIdx.x];
  if ((uint32_t)tile.x >= (uint32_t)p.G) return;  // past the last tile
  if (tile.y < 0 || tile.z <= 0 || tile.z > kLowRows || tile.y > p.M - tile.z) return;  // not a plan's
  const float sc = p.scale[tile.x];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, kg = lane >> 4;
  const int r0 = blockIdx.y * RT * 16;
  const int k0 = blockIdx.z * p.kpart, k1 = min(k0 + p.kpart, p.K), iters = (k1 - k0 + BK - 1) / BK;
  const __amdgpu_buffer_rsrc_t rx = bytes_rsrc(p.x, (uint32_t)((p.M - 1) * p.x_s + p.K) * E);
  const __amdgpu_buffer_rsrc_t ra = bytes_rsrc(p.a + (int64_t)tile.x * p.r * p.K, (uint32_t)p.r * p.K * E);
  // chunk c of a stage: row c / CH of [x rows ; A rows], LDS position c % CH; rows past the
  // tile's and ranks past the last are loaded again
  uint32_t off[LPS], col[LPS];
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const int c = (i * kLowWaves + wave) * 64 + lane;
    const int r = c / CH, pos = c % CH;
    col[i] = ((pos & ~7) | ((pos ^ r) & 7)) * V;
    off[i] = r < kLowRows ? (uint32_t)(plan_row(p, tile.y + min(r, tile.z - 1)) * p.x_s) * E
                          : (uint32_t)(min(r0 + r - kLowRows, p.r - 1) * p.K) * E;
  }
  auto issue = [&](int st, int k) {
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const int base = (i * kLowWaves + wave) * 64;
      const uint32_t at = k + (int)col[i] < k1 ? (uint32_t)k + col[i] : (uint32_t)k0;
      load_lds16(base < kLowRows * CH ? rx : ra, smem + st * kStage + base * 16, off[i] + at * E, 0);
    }
  };
  f32x4_t acc[RT][2];
#pragma unroll
  for (int j = 0; j < RT; ++j) acc[j][0] = acc[j][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < iters) issue(s, k0 + s * BK);
  int st = 0;
  for (int it = 0; it < iters; ++it) {
    if (it + S - 2 < iters)
      wait_vm<(S - 2) * LPS>();
    else
      wait_vm<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (it + S - 1 < iters) issue(st == 0 ? S - 1 : st - 1, k0 + (it + S - 1) * BK);
    if (k0 + it * BK + wave * COLS < k1) {
      const int ch = wave * 4 + kg;
      auto frag = [&](int r) { return *reinterpret_cast<const u32x4*>(smem + st * kStage + r * ROW + ((ch & ~7) | ((ch ^ r) & 7)) * 16); };
      const u32x4 xf[2] = {frag(l16), frag(16 + l16)};
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const u32x4 af = frag(kLowRows + j * 16 + l16);
        acc[j][0] = MmaA<ST>::step(af, xf[0], acc[j][0]);
        acc[j][1] = MmaA<ST>::step(af, xf[1], acc[j][1]);
      }
    }
    st = st == S - 1 ? 0 : st + 1;
  }
  __syncthreads();  // the stages are read
  f32x4_t* const red = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int m = 0; m < 2; ++m) red[((wave * RT + j) * 2 + m) * 64 + lane] = acc[j][m];
  __syncthreads();
  const int row = (wave & 1) * 16 + l16, c = r0 + (wave >> 1) * 16 + kg * 4;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  if (wave < 2 * RT) {
    v = red[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < kLowWaves; ++w) v += red[(w * RT * 2 + wave) * 64 + lane];
  }
  RowUnit u{1.f, 1.f};
  if constexpr (kUnits<ST>) {  // ranks past the last are the last again, and no larger
    float m = largest_of_row(v, sc);
    if constexpr (RT > 1) {
      float* const most = reinterpret_cast<float*>(smem + kRed);
      if (wave < 2 * RT && kg == 0) most[wave * 16 + l16] = m;
      __syncthreads();
      if (wave < 2 * RT) {
#pragma unroll
        for (int j = 0; j < RT; ++j) m = fmaxf(m, most[(2 * j + (wave & 1)) * 16 + l16]);
      }
    }
    u = row_unit(m);
  }
  if (wave >= 2 * RT || row >= tile.z) return;
  ST* const hp = p.h + (tile.y + row) * (int64_t)(low_row<ST>(p.r, p.parts) / E);
  if (kUnits<ST> && wave < 2 && kg == 0) reinterpret_cast<float*>(hp + 2 * p.r * p.parts)[blockIdx.z * gridDim.y + blockIdx.y] = u.up;
  if (c < p.r) store_low<ST>(v, sc, u.down, hp + blockIdx.z * (E == 4 ? p.r : 2 * p.r) + c, p.r);  // r is a multiple of 8, c of 4
}

// whether every sum is finite: an infinity or NaN times zero is a NaN
template <int TM, int TN>
__device__ static inline bool all_finite(const f32x4_t (&acc)[TM][TN]) {
  float z = 0.f;
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) z = fmaf(acc[m][n][e], 0.f, z);
  return z == 0.f;
}

// add_low where an infinity or NaN is among the operands: where only some of 16 rows have
// an adapter its product is taken for all of them and kept for those, so that what a row
// gets depends on its own adapter alone, and in the same order of sums, so that the rows
// without them keep their bits.
template <typename ST, int TM, int TN, int WK, bool LDS, bool FIT, typename Fit>
__device__ static inline void add_low_apart(const AdK<ST>& p, const int (&id)[TM], int pos0, int c0, int wk, int lane,
                                            Fit fit, f32x4_t (&acc)[TM][TN]) {
  constexpr int V = Tr<ST>::VEC;
  const int l16 = lane & 15, kg = lane >> 4;
  const int hs = low_row<ST>(p.r, p.parts) / sizeof(ST);
  const LowOrder o = low_order<ST, LDS>(p.r, p.parts);
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
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      has[m] = __ballot(id[m] == g);
      left[m] &= ~has[m];
    }
    if (WK > 1 && turn != wk) continue;
    const ST* const bp = p.b + ((int64_t)g * p.N + c0 + l16) * p.r;
    auto b_of = [&](int n, int q, int end) { return q < end ? ld16(bp + (int64_t)n * 16 * p.r + b_chunk<ST>(q, p.r) * V) : zero; };
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      if (has[m] == 0) continue;
      f32x4_t d[TN];
#pragma unroll
      for (int n = 0; n < TN; ++n) d[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      for (int q0 = 0; q0 < o.width; q0 += o.block) {
        const int end = min(q0 + o.block, o.width);
        for (int q = q0 + kg; q - kg < end; q += 4)
          for (int c = 0; c < o.copies; ++c) {
            u32x4 hf = q < end ? ld16(hp[m] + (c * o.width + q) * V) : zero;
            if constexpr (FIT) hf = fit(m, piece_of(o, p.r, c, min(q, end - 1)), hf);
#pragma unroll
            for (int n = 0; n < TN; ++n) d[n] = MmaA<ST>::step(b_of(n, q, end), hf, d[n]);
          }
      }
      if (id[m] == g) {
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] += d[n];
      }
    }
  }
}

// acc[m][n] += h B^T for TM x TN products of rows pos0 + 16 m and columns c0 + 16 n, over
// chunks qa .. qb of the copies of h, summed over the adapters among the rows (of these,
// part `wk` of WK), each with the other adapters' rows of h read as zero.  Work items of one
// adapter and 4 chunks of B, DEP items' loads on their way: a wave with few rows has up to
// 16 adapters a product, and one by one each would cost a round trip to memory (0.8 us).
// LDS: the chunks of h are at hs, kLowRow bytes a row from local row lr0 on, once `ready` has
// waited for them; else they are read with B's.  FIT: fit(m, piece, chunk) brings a chunk of h
// to its row's units.  A zero row of h times an infinity in B is a NaN in another adapter's
// rows: the caller makes sums that are not finite again.
template <typename ST, int TM, int TN, int WK, int DEP, bool LDS, bool FIT, typename Ready, typename Fit>
__device__ static inline void add_low(const AdK<ST>& p, const int (&id)[TM], int pos0, int c0, int wk, int lane, const unsigned char* hs,
                                      int lr0, const LowOrder o, int qa, int qb, Ready ready, Fit fit, f32x4_t (&acc)[TM][TN]) {
  constexpr uint32_t E = sizeof(ST);
  const int l16 = lane & 15, kg = lane >> 4;
  const uint32_t hrow = low_row<ST>(p.r, p.parts), brow = p.r * E;
  const __amdgpu_buffer_rsrc_t rh = bytes_rsrc(p.h, (uint32_t)p.M * hrow);
  uint64_t left[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) left[m] = __ballot(id[m] >= 0);
  struct Item {
    u32x4 bf[TN], hf[LDS ? 1 : TM];
    uint32_t rows;  // bit m: rows 16 m have the adapter; 0: no item
    int g, q;
  };
  int g = -1, q0 = 0, turn = 0;
  uint32_t rows = 0;
  auto next = [&](Item& it) {
    q0 += 4;
    if (g < 0 || q0 >= qb) {
      q0 = qa;
      bool mine = false;
      do {
        g = -1;
        rows = 0;
#pragma unroll
        for (int m = TM - 1; m >= 0; --m)
          if (left[m]) g = __builtin_amdgcn_readlane(id[m], __builtin_ctzll(left[m]));
        if (g < 0) break;
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          const uint64_t has = __ballot(id[m] == g);
          left[m] &= ~has;
          rows |= has ? 1u << m : 0u;
        }
        mine = WK == 1 || turn == wk;
        turn = turn == WK - 1 ? 0 : turn + 1;
      } while (!mine);
    }
    it.rows = rows;
    it.g = g;
    it.q = q0;
    if (!rows) return;
    const int q = q0 + kg;
    const __amdgpu_buffer_rsrc_t rb = bytes_rsrc(p.b + (int64_t)g * p.N * p.r, (uint32_t)p.N * brow);
    const uint32_t bo = q < qb ? (uint32_t)(c0 + l16) * brow + (uint32_t)b_chunk<ST>(q, p.r) * 16u : kNowhere;
#pragma unroll
    for (int n = 0; n < TN; ++n) it.bf[n] = load16(rb, bo + (uint32_t)(n * 16) * brow);
    if constexpr (!LDS) {
#pragma unroll
      for (int m = 0; m < TM; ++m)
        it.hf[m] = load16(rh, q < qb && id[m] == g ? (uint32_t)(pos0 + m * 16 + l16) * hrow + (uint32_t)q * 16u : kNowhere);
    }
  };
  Item it[DEP];
#pragma unroll
  for (int d = 0; d < DEP; ++d) next(it[d]);
  ready();
  for (bool more = true; more;) {
#pragma unroll
    for (int d = 0; d < DEP; ++d) {
      if (!it[d].rows) {
        more = false;
        break;
      }
      for (int c = 0; c < (LDS ? o.copies : 1); ++c) {
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          if (!(it[d].rows >> m & 1)) continue;
          u32x4 hf = {0u, 0u, 0u, 0u};
          if constexpr (LDS) {
            const int r = lr0 + m * 16 + l16, ch = c * o.block + it[d].q - qa + kg;
            if (id[m] == it[d].g && it[d].q + kg < qb) hf = *reinterpret_cast<const u32x4*>(hs + r * kLowRow + ((ch & ~7) | ((ch ^ r) & 7)) * 16);
          } else {
            hf = it[d].hf[m];
          }
          if constexpr (FIT) hf = fit(m, piece_of(o, p.r, c, min(it[d].q + kg, qb - 1)), hf);  // zeros stay zeros
#pragma unroll
          for (int n = 0; n < TN; ++n) acc[m][n] = MmaA<ST>::step(it[d].bf[n], hf, acc[m][n]);
        }
      }
      next(it[d]);
    }
  }
}

// SiLU with the hardware's reciprocal (1 ulp): a full division is 11 more instructions a
// value, 4 us of a launch of 3584 x 4096 outputs.  The reciprocal gives 0 for results below
// 2^-126, where v / (1 + exp(-v)) is still a normal number (v from -87.3 to -88.7): it is taken
// of 2^-8 of the divisor and the factor put back, 0.2 us of that launch.
template <int SILU>
__device__ static inline float ad_act(float v) {
  if constexpr (SILU) return v * (__builtin_amdgcn_rcpf(fmaf(__expf(-v), 0x1p-8f, 0x1p-8f)) * 0x1p-8f);
  return v;
}

// A tile's output: sums of the parts of K, bias and activation, then through LDS (smem,
// free when every wave is here) to whole 16-byte chunks of the rows that `ord` names.
template <typename ST, int BM, int BN, int WM, int WN, int WK, int TM, int TN, int SILU>
__device__ static inline void store_out(const AdK<ST>& p, unsigned char* smem, f32x4_t (&acc)[TM][TN], const int32_t* ord, int row0, int n0,
                                        int wave, int lane) {
  constexpr int E = sizeof(ST), V = 16 / E;
  constexpr int OS = BN + V;  // LDS row stride of the staged output
  const int l16 = lane & 15, kg = lane >> 4;
  const int wk = wave / (WM * WN), wm = (wave / WN) % WM, wn = wave % WN;
  sum_parts<BM, BN, WM * WN, WK>(smem, BM * OS * E, acc, wave, lane);
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
        ST* const o = os + ((wm * TM + m) * 16 + l16) * OS + c;
        if constexpr (E == 4)
          *reinterpret_cast<u32x4*>(o) = Tr<float>::pack(f);
        else
          *reinterpret_cast<u32x2*>(o) = pack4<ST>(f);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BM * BN / V; i += 64 * WM * WN * WK) {
    const int r = i / (BN / V), c = (i % (BN / V)) * V;
    if (row0 + r < p.M) st16(p.out + (int64_t)ord[r] * p.out_s + n0 + c, *reinterpret_cast<const u32x4*>(os + r * OS + c));
  }
}

// The product with W: BM x BN outputs a workgroup, both operands staged in LDS as in
// lin_tile_kernel, the rows of x and of the output those that the plan's order names.
//
// The adapters' part comes first (add_low), while the first stages are on their way.  Tiles
// of 64 rows and more (kStaged) have their rows of h in LDS for it, 16 chunks a row in the
// stage that the main loop fills last: a byte of h is then loaded once a workgroup, B goes
// from memory to the waves that multiply it.  Tiles of fewer rows read h as they read B: LDS
// would save nothing, a wave column or two share it.
//
// Bound by the round trips of the K loop: one stage of 64 KB a CU is on its way for the
// largest tiles, matrix cores busy 29% of the time.  bf16: 3584 rows 1024 -> 4096 in 37.8 us
// (795 TFLOP/s) without adapters and SiLU, 840 rows 4096 -> 1024 in 20.7 us with 12 adapters
// of rank 32, 61 rows with an adapter of rank 16 each in 6.5 us.
// FIT: rows of h in several pieces that have units (fp16).  A form of its own: 3584 rows 1024 ->
// 4096 of rank 128 take 66 us so and 68 with a branch in the loop of h B^T.
template <typename ST, int BM, int BN, int WM, int WN, int WK, int BK, int S, int SILU, bool FIT>
__global__ void __launch_bounds__(64 * WM * WN * WK) adapter_tile_kernel(const AdK<ST> p) {
#pragma clang fp contract(off)
  constexpr int NW = WM * WN * WK;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int E = sizeof(ST), V = 16 / E;
  constexpr int ROW = BK * E, CH = ROW / 16;  // bytes and 16-byte chunks of a row's stage
  constexpr int kStage = (BM + BN) * ROW;
  constexpr int LPS = kStage / 1024 / NW;
  static_assert(ROW % 128 == 0, "the permutation stays within a row's stage: whole groups of 8 chunks");
  static_assert(kStage % (1024 * NW) == 0 && (BM * CH) % 64 == 0, "whole waves of chunks");
  constexpr int KS = CH / 4 / WK;  // steps of 4 chunks a lane group a wave does a stage
  constexpr int OS = BN + V;       // LDS row stride of the staged output
  constexpr int kOut = BM * OS * E;
  constexpr int kRed = WK > 1 ? (WK - 1) * BM * BN * 4 : 0;
  constexpr int kSmem = S * kStage > kOut + kRed ? S * kStage : kOut + kRed;
  constexpr bool kStaged = CH == 8;
  // one LDS object: with a second one the compiler keeps them apart and waits for every
  // load to LDS in flight before an operand read
  __shared__ __align__(16) unsigned char smem[kSmem + BM * (!kUnits<ST> || !kStaged ? 8 : FIT ? 8 + 8 * kMaxUnits : 8 + 4 * kMaxUnits)];
  int32_t* const ord = reinterpret_cast<int32_t*>(smem + kSmem);
  int32_t* const sid = ord + BM;
  u32x4* const units = reinterpret_cast<u32x4*>(sid + BM);          // fp16, staged: the units of a row of h
  uint32_t* const ratio = reinterpret_cast<uint32_t*>(units + BM);  // FIT: [kMaxUnits][BM] of its pieces to the largest

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, kg = lane >> 4;
  const int wk = wave / (WM * WN), wm = (wave / WN) % WM, wn = wave % WN;
  int mt_i, nt_i;
  xcd_tile(p.mtiles, p.xm, mt_i, nt_i);
  const int row0 = mt_i * BM, n0 = nt_i * BN;

  const uint32_t hrow = low_row<ST>(p.r, p.parts);
  const __amdgpu_buffer_rsrc_t rh = bytes_rsrc(p.h, (uint32_t)p.M * hrow);
  // fp16: where a row of h has its units
  auto units_at = [&](int pos) { return pos < p.M ? (uint32_t)pos * hrow + (uint32_t)p.r * 4u * p.parts : kNowhere; };
  auto most_of = [&](u32x4 u) {
    float most = __uint_as_float(u[0]);
    if constexpr (FIT) {
#pragma unroll
      for (int j = 1; j < kMaxUnits; ++j) most = j < p.units ? fmaxf(most, __uint_as_float(u[j])) : most;
    }
    return most;
  };
  // positions past the last row read the last row, have no adapter and store nothing
  for (int i = threadIdx.x; i < BM; i += 64 * NW) {
    ord[i] = plan_row(p, row0 + i);
    const int g = p.ids[min(row0 + i, p.M - 1)];
    sid[i] = row0 + i < p.M && (uint32_t)g < (uint32_t)p.G ? g : -1;
  }
  __syncthreads();
  int id[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) id[m] = sid[(wm * TM + m) * 16 + l16];
  const __amdgpu_buffer_rsrc_t rx = bytes_rsrc(p.x, (uint32_t)((p.M - 1) * p.x_s + p.K) * E);
  const __amdgpu_buffer_rsrc_t rw = bytes_rsrc(p.w, (uint32_t)((p.N - 1) * p.w_s + p.K) * E);
  // chunk c of a stage: row c / CH of [x rows ; w rows], LDS position c % CH
  uint32_t off[LPS];
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const int c = (i * NW + wave) * 64 + lane;
    const int r = c / CH, pos = c % CH;
    const int ch = (pos & ~7) | ((pos ^ r) & 7);
    off[i] = r < BM ? (uint32_t)(ord[r] * p.x_s + ch * V) * E : (uint32_t)((n0 + r - BM) * p.w_s + ch * V) * E;
  }
  auto issue = [&](int st, int k) {
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const int base = (i * NW + wave) * 64;
      load_lds16(base < BM * CH ? rx : rw, smem + st * kStage + base * 16, off[i], k * E);
    }
  };
  f32x4_t acc[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int n = 0; n < TN; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int st) {
    const unsigned char* xs = smem + st * kStage;
    const unsigned char* ws = xs + BM * ROW;
    u32x4 xf[KS][TM], wf[KS][TN];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ch = (wk * KS + s) * 4 + kg;
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        const int r = (wn * TN + n) * 16 + l16;
        wf[s][n] = *reinterpret_cast<const u32x4*>(ws + r * ROW + ((ch & ~7) | ((ch ^ r) & 7)) * 16);
      }
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const int r = (wm * TM + m) * 16 + l16;
        xf[s][m] = *reinterpret_cast<const u32x4*>(xs + r * ROW + ((ch & ~7) | ((ch ^ r) & 7)) * 16);
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = MmaA<ST>::step(wf[s][n], xf[s][m], acc[m][n]);
    // One workgroup a CU has no other to fill the matrix cores while it reads LDS: operand
    // reads one between two matrix instructions (3584 rows 1024 -> 4096: 37.8 us, 42.4 with a
    // step's reads before its products; 128 x 128 tiles gain nothing, 64 x 64 lose 5%).
    if constexpr (BM == 256) {
      __builtin_amdgcn_sched_group_barrier(0x100, TN + 2, 0);
#pragma unroll
      for (int i = 0; i < KS * (TM + TN) - TN - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
  };
  auto wait = [&](bool last) {
    if (!last)
      wait_vm<(S - 2) * LPS>();
    else
      wait_vm<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  const int iters = p.K / BK;
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < iters) issue(s, s * BK);
  const int pos0 = row0 + wm * TM * 16, c0 = n0 + wn * TN * 16;
  const LowOrder o = low_order<ST, kStaged>(p.r, p.parts);
  // fp16: the sums to what they stand for (nothing is written for rows without an adapter)
  auto in_ones = [&](auto up_of) {
    if constexpr (kUnits<ST>) {
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const float u = up_of(m);
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] *= u;
      }
    }
  };
  auto again = [&](auto fit) {  // an infinity or NaN is among the operands
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
      for (int n = 0; n < TN; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    add_low_apart<ST, TM, TN, WK, kStaged, FIT>(p, id, pos0, c0, wk, lane, fit, acc);
  };
  if constexpr (kStaged) {
    constexpr int LPH = BM * kLowRow / 1024 / NW;
    static_assert(BM * kLowRow <= kStage && BM * kLowRow % (1024 * NW) == 0, "h fits a stage");
    unsigned char* const hs = smem + (S - 1) * kStage;
    auto meet = [&]() {  // every wave's loads to LDS are in, its reads done
      wait_vm<0>();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    if constexpr (kUnits<ST>) {
      static_assert(BM <= 64 * NW, "64 rows a wave");
      if (wave < BM / 64) load_lds16(rh, reinterpret_cast<unsigned char*>(units + wave * 64), units_at(row0 + wave * 64 + lane), 0);
    }
    bool first = true;
    auto ready = [&]() {
      meet();
      if (FIT && first) {
        if (threadIdx.x < BM) {
          const u32x4 u = units[threadIdx.x];
          const float most = most_of(u);
#pragma unroll
          for (int j = 0; j < kMaxUnits; ++j) ratio[j * BM + threadIdx.x] = unit_ratio(__uint_as_float(u[j]), most);
          units[threadIdx.x][0] = __float_as_uint(most);
        }
        meet();
      }
      first = false;
    };
    const int row = wm * TM * 16 + l16;
    auto fit = [&](int m, int piece, u32x4 h) { return to_unit(h, ratio[piece * BM + row + m * 16]); };
    auto up_of = [&](int m) { return id[m] >= 0 ? __uint_as_float(units[row + m * 16][0]) : 1.f; };
    for (int qa = 0; qa < o.width; qa += o.block) {
      if (qa > 0) meet();  // the chunks before are read
#pragma unroll
      for (int i = 0; i < LPH; ++i) {
        const int c = (i * NW + wave) * 64 + lane, r = c / kLowChunks, pos = c % kLowChunks;
        const int ch = (pos & ~7) | ((pos ^ r) & 7), copy = ch >> o.shift, q = qa + (ch & (o.block - 1));
        const uint32_t at = (uint32_t)(row0 + r) * hrow + (uint32_t)(copy * o.width + q) * 16u;
        load_lds16(rh, hs + (i * NW + wave) * 1024, row0 + r < p.M && q < o.width ? at : kNowhere, 0);
      }
      // 256 x 256: 3 items, with 4 the registers spill (r 16: 61 us for 54)
      constexpr int DEP = TM * TN >= 32 ? 3 : 4;
      add_low<ST, TM, TN, WK, DEP, true, FIT>(p, id, pos0, c0, wk, lane, hs, wm * TM * 16, o, qa, min(qa + o.block, o.width), ready, fit, acc);
    }
    if (__ballot(!all_finite(acc))) again(fit);
    in_ones(up_of);
  } else {
    u32x4 u[TM];
    if constexpr (kUnits<ST>) {
#pragma unroll
      for (int m = 0; m < TM; ++m) u[m] = load16(rh, units_at(pos0 + m * 16 + l16));
    }
    auto fit = [&](int m, int piece, u32x4 h) {
      uint32_t own = u[m][0];
#pragma unroll
      for (int j = 1; j < kMaxUnits; ++j) own = piece == j ? u[m][j] : own;
      return to_unit(h, unit_ratio(__uint_as_float(own), most_of(u[m])));
    };
    auto up_of = [&](int m) { return id[m] >= 0 ? most_of(u[m]) : 1.f; };
    add_low<ST, TM, TN, WK, 4, false, FIT>(p, id, pos0, c0, wk, lane, nullptr, 0, o, 0, o.width, []() {}, fit, acc);
    if (__ballot(!all_finite(acc))) again(fit);
    in_ones(up_of);
  }
  int st = 0;
  for (int it = 0; it < iters; ++it) {
    wait(it + S - 2 >= iters);
    if (it + S - 1 < iters) issue(st == 0 ? S - 1 : st - 1, (it + S - 1) * BK);
    multiply(st);
    st = st == S - 1 ? 0 : st + 1;
  }
  __syncthreads();
  store_out<ST, BM, BN, WM, WN, WK, TM, TN, SILU>(p, smem, acc, ord, row0, n0, wave, lane);
}

// Few rows, in one launch: 16 rows x BN outputs a workgroup, their x whole in LDS, where h of
// the tile's adapters is made while the first stages of W are on their way.  Every
// workgroup of a row tile makes the same h again and reads its adapters' A, which is less
// than a launch of its own (3.3 us of the host's, 4 of the GPU's) while a tile has few
// adapters.  RW: bytes of a row of x.
template <typename ST, int RW, int RT, int BN, int WN, int WK, int BKB, int S, int SILU>
__global__ void __launch_bounds__(64 * WN * WK) adapter_few_kernel(const AdK<ST> p) {
#pragma clang fp contract(off)
  // fp16: h in fp32 and B widened to it for the fp32 instructions, few here; h keeps its range
  // without units, whose maximum would be in the chain (256 rows 512 -> 2048, r 16: 7.7 us so,
  // 8.3 with units)
  using HT = std::conditional_t<kUnits<ST>, float, ST>;
  using BF = std::conditional_t<kUnits<ST>, u32x2, u32x4>;
  constexpr int E = sizeof(ST), V = 16 / E, COLS = MmaA<ST>::COLS;
  constexpr int K = RW / E, BK = BKB / E, CH = BKB / 16;
  constexpr int NW = WN * WK, BM = 16, TN = BN / WN / 16;
  constexpr int kAct = BM * RW, kStage = BN * BKB;
  constexpr int LPS = kStage / 1024 / NW, LPX = kAct / 1024 / NW;
  constexpr int KS = CH / 4 / WK, iters = K / BK;
  static_assert(NW == 8 && BKB % 128 == 0 && RW % BKB == 0 && kStage % (1024 * NW) == 0 && kAct % (1024 * NW) == 0 && KS > 0, "whole waves of chunks");
  constexpr int U = 4, AS = K / COLS / NW;  // steps of K a wave does for h, U of them on their way
  static_assert(K % (COLS * NW) == 0, "whole steps a wave");
  constexpr int OS = BN + V, kOut = BM * OS * E, kRed = (WK - 1) * BM * BN * 4;
  constexpr int kLow = NW * RT * 1024, kH = BM * RT * 64;
  constexpr int kMain = kAct + S * kStage > kOut + kRed ? kAct + S * kStage : kOut + kRed;
  __shared__ __align__(16) unsigned char smem[kMain + kLow + kH + BM * 8];
  f32x4_t* const red = reinterpret_cast<f32x4_t*>(smem + kMain);
  unsigned char* const hs = smem + kMain + kLow;  // [16] rows of h
  int32_t* const ord = reinterpret_cast<int32_t*>(hs + kH);
  int32_t* const sid = ord + BM;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, kg = lane >> 4;
  const int wk = wave / WN, wn = wave % WN;
  int mt_i, nt_i;
  xcd_tile(p.mtiles, p.xm, mt_i, nt_i);
  const int row0 = mt_i * BM, n0 = nt_i * BN;
  if (threadIdx.x < BM) {
    const int pos = row0 + threadIdx.x;
    ord[threadIdx.x] = plan_row(p, pos);
    const int g = p.ids[min(pos, p.M - 1)];
    sid[threadIdx.x] = pos < p.M && (uint32_t)g < (uint32_t)p.G ? g : -1;
  }
  __syncthreads();
  const int id = sid[l16];
  const __amdgpu_buffer_rsrc_t rx = bytes_rsrc(p.x, (uint32_t)((p.M - 1) * p.x_s + p.K) * E);
  const __amdgpu_buffer_rsrc_t rw = bytes_rsrc(p.w, (uint32_t)((p.N - 1) * p.w_s + p.K) * E);
  unsigned char* const ring = smem + kAct;
#pragma unroll
  for (int i = 0; i < LPX; ++i) {
    const int c = (i * NW + wave) * 64 + lane, r = c / (RW / 16), pos = c % (RW / 16);
    load_lds16(rx, smem + (i * NW + wave) * 1024, (uint32_t)(ord[r] * p.x_s) * E + (uint32_t)(((pos & ~7) | ((pos ^ r) & 7)) * 16), 0);
  }
  uint32_t off[LPS];
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const int c = (i * NW + wave) * 64 + lane, r = c / CH, pos = c % CH;
    off[i] = (uint32_t)((n0 + r) * p.w_s) * E + (uint32_t)(((pos & ~7) | ((pos ^ r) & 7)) * 16);
  }
  auto issue = [&](int st, int it) {
#pragma unroll
    for (int i = 0; i < LPS; ++i) load_lds16(rw, ring + st * kStage + (i * NW + wave) * 1024, off[i], it * BKB);
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s)
    if (s < iters) issue(s, s);
  auto x_frag = [&](int ch) { return *reinterpret_cast<const u32x4*>(smem + l16 * RW + ((ch & ~7) | ((ch ^ l16) & 7)) * 16); };
  auto meet = [&]() {  // the waves' LDS stores are done; loads to LDS stay in flight
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f32x4_t acc[1][TN];
#pragma unroll
  for (int n = 0; n < TN; ++n) acc[0][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const uint32_t arow = (uint32_t)p.r * E, chunks = p.r >> 2;
  uint32_t left = (uint32_t)(__ballot(id >= 0) & 0xffff);
  int turn = 0;
  bool first = true;
  while (left) {
    const int g = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    const bool mine = id == g;
    left &= ~(uint32_t)(__ballot(mine) & 0xffff);
    const __amdgpu_buffer_rsrc_t ra = bytes_rsrc(p.a + (int64_t)g * p.r * K, arow * K);
    const __amdgpu_buffer_rsrc_t rb = bytes_rsrc(p.b + (int64_t)g * p.N * p.r, (uint32_t)p.N * arow);
    f32x4_t h[RT];
#pragma unroll
    for (int j = 0; j < RT; ++j) h[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s0 = 0; s0 < AS; s0 += U) {
      u32x4 af[U][RT];
#pragma unroll
      for (int u = 0; u < U && s0 + u < AS; ++u)
#pragma unroll
        for (int j = 0; j < RT; ++j)
          af[u][j] = load16(ra, (uint32_t)(min(j * 16 + l16, p.r - 1) * K + ((s0 + u) * NW + wave) * COLS) * E + kg * 16u);
      if (first) {  // the rows of x are in for every wave
        wait_vm<0>();
        meet();
        first = false;
      }
#pragma unroll
      for (int u = 0; u < U && s0 + u < AS; ++u)
#pragma unroll
        for (int j = 0; j < RT; ++j) h[j] = MmaA<ST>::step(af[u][j], x_frag(((s0 + u) * NW + wave) * 4 + kg), h[j]);
    }
    // this adapter's B for the wave's columns, on its way while the sums meet
    BF bf[RT][TN];
    const bool turn_mine = turn == wk;
    turn = turn == WK - 1 ? 0 : turn + 1;
    if (turn_mine) {
#pragma unroll
      for (int q = 0; q < RT; ++q)
#pragma unroll
        for (int n = 0; n < TN; ++n) {
          const uint32_t c = q * 4 + kg;  // 16 ranks a step
          const uint32_t row = (uint32_t)(n0 + (wn * TN + n) * 16 + l16) * arow;
          if constexpr (kUnits<ST>)
            bf[q][n] = load8(rb, c < chunks ? row + c * 8u : kNowhere);
          else
            bf[q][n] = load16(rb, c < chunks ? row + (uint32_t)b_chunk<ST>(c, p.r) * 16u : kNowhere);
        }
    }
#pragma unroll
    for (int j = 0; j < RT; ++j) red[(wave * RT + j) * 64 + lane] = h[j];
    meet();
    if (wave < RT) {
      f32x4_t v = red[wave * 64 + lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) v += red[(w * RT + wave) * 64 + lane];
      const int c = wave * 16 + kg * 4;
      if (mine && c < p.r) store_low<HT>(v, p.scale[g], 1.f, reinterpret_cast<HT*>(hs + l16 * (RT * 64)) + c, p.r);
    }
    meet();
    if (turn_mine) {
      f32x4_t d[TN];
#pragma unroll
      for (int n = 0; n < TN; ++n) d[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        const uint32_t c = q * 4 + kg;
        u32x4 hf = {0u, 0u, 0u, 0u};
        if (mine && c < chunks) hf = *reinterpret_cast<const u32x4*>(hs + l16 * (RT * 64) + c * 16);
#pragma unroll
        for (int n = 0; n < TN; ++n) d[n] = MmaA<HT>::step(wide(bf[q][n]), hf, d[n]);
      }
      // columns (rows of the batch) are independent: kept for the adapter's own rows
#pragma unroll
      for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][n][e] = mine ? d[n][e] : acc[0][n][e];
    }
  }

  int st = 0;
#pragma unroll 1
  for (int it = 0; it < iters; ++it) {
    if (!first && it + S - 2 < iters)
      wait_vm<(S - 2) * LPS>();
    else
      wait_vm<0>();
    first = false;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (it + S - 1 < iters) issue(st == 0 ? S - 1 : st - 1, it + S - 1);
    const unsigned char* ws = ring + st * kStage;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int ch = (wk * KS + s) * 4 + kg;
      const u32x4 xf = x_frag(it * CH + ch);
#pragma unroll
      for (int n = 0; n < TN; ++n) {
        const int r = (wn * TN + n) * 16 + l16;
        const u32x4 wf = *reinterpret_cast<const u32x4*>(ws + r * BKB + ((ch & ~7) | ((ch ^ r) & 7)) * 16);
        acc[0][n] = MmaA<ST>::step(wf, xf, acc[0][n]);
      }
    }
    st = st == S - 1 ? 0 : st + 1;
  }
  __syncthreads();
  store_out<ST, BM, BN, 1, WN, WK, 1, TN, SILU>(p, smem, acc, ord, row0, n0, wave, lane);
}

namespace {

// workgroups over the ranks, 64 of them each
int low_blocks(int r) { return (r + 63) / 64; }

// Parts of K that x A^T is split into: two, of 1024 columns or more, while there are at most
// 256 workgroups (one a CU): 32 x 2 rows 4096 -> 1024 take 16.3 us so and 18.1 in one part; the
// product with B then takes twice the steps (840 rows of rank 64: 38.5 and 38.7; in four
// parts 43.3).
int k_parts(int64_t tiles, int r, int64_t k) { return k >= 2048 && tiles * low_blocks(r) * 2 <= 256 ? 2 : 1; }

template <typename ST>
int launch_low(const AdK<ST>& k, int max_tiles, hipStream_t s) {
  const dim3 grid((unsigned)max_tiles, (unsigned)low_blocks(k.r), (unsigned)k.parts), block(64 * kLowWaves);
  if (k.r <= 16)
    hipLaunchKernelGGL((adapter_low_kernel<ST, 1, 4>), grid, block, 0, s, k);
  else if (k.r <= 32)
    hipLaunchKernelGGL((adapter_low_kernel<ST, 2, 4>), grid, block, 0, s, k);
  else
    hipLaunchKernelGGL((adapter_low_kernel<ST, 4, 3>), grid, block, 0, s, k);
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
  // BK columns of 16-bit types; of fp32 half as many, the same bytes
  constexpr int B = BK * 2 / (int)sizeof(ST);
  if (kUnits<ST> && k.units > 1)
    hipLaunchKernelGGL((adapter_tile_kernel<ST, BM, BN, WM, WN, WK, B, S, SILU, kUnits<ST>>), grid, dim3(64 * WM * WN * WK), 0, s, k);
  else
    hipLaunchKernelGGL((adapter_tile_kernel<ST, BM, BN, WM, WN, WK, B, S, SILU, false>), grid, dim3(64 * WM * WN * WK), 0, s, k);
  return check_launch("pk_adapter_linear");
}

// The forms of the product and what a launch of each takes: `a` us and `s` us a 1024
// columns for a workgroup alone on its CU, `m` of the latter for each further one beside
// it (`occ` fit), again a - 2 for each further round, and `e` us for a step of the adapters'
// part: a run of rows with one adapter in a tile, 16 ranks of it.
// Fitted to launches in a graph, 1 - 8192 rows (fp32 1800), K and N 512 - 4096, ranks 16 to 64,
// from one adapter to one for every second row.  Over 256 such sizes of 16-bit types, and 90 of
// fp32, the cheapest by it takes 0.3 - 0.7% more than the fastest form on the mean and 12% at the
// worst.  How many adapters the rows have is not known on the host; the plan's tiles bound it.
struct Form {
  int bm, bn, occ;
  bool staged;
};
struct FormCost {
  float a, s, m, e;
};
constexpr Form kForms[] = {{16, 16, 4, false}, {16, 32, 3, false}, {32, 32, 2, false},  {32, 64, 2, false},
                           {64, 64, 2, true},  {64, 128, 2, true}, {128, 128, 2, true}, {256, 256, 1, true}};
constexpr FormCost kCostBf16[] = {{3.40f, 1.89f, 0.20f, 0.03f},  {3.43f, 2.33f, 0.23f, 0.05f},  {4.15f, 2.69f, 0.36f, 0.06f},
                                  {3.22f, 5.26f, 0.17f, 0.21f},  {3.78f, 4.51f, 0.44f, 0.06f},  {2.57f, 13.12f, 0.15f, 0.13f},
                                  {6.43f, 11.02f, 0.26f, 0.19f}, {9.04f, 20.58f, 0.f, 0.25f}};
// (64 x 128 tiles of fp16 are compiled to a faster loop: 3584 rows 4096 -> 1024, rank 16, 52.5 us, 58.4 in
// 128 x 128; bf16 62.8 and 58.1)
constexpr FormCost kCostF16[] = {{3.40f, 1.89f, 0.20f, 0.03f},  {3.43f, 2.33f, 0.23f, 0.05f},  {4.15f, 2.69f, 0.36f, 0.06f},
                                 {3.00f, 5.26f, 0.17f, 0.21f},  {3.78f, 5.14f, 0.44f, 0.06f},  {2.37f, 10.05f, 0.15f, 0.12f},
                                 {5.88f, 11.65f, 0.26f, 0.19f}, {9.04f, 20.58f, 0.f, 0.25f}};
// fp32 (256 x 256 outputs of it do not fit LDS)
constexpr FormCost kCost32[] = {{3.53f, 4.16f, 0.22f, 0.03f},  {3.75f, 5.68f, 0.20f, 0.05f},  {3.61f, 7.45f, 0.28f, 0.07f},
                                {2.56f, 15.91f, 0.22f, 0.15f}, {4.95f, 19.60f, 0.53f, 0.15f}, {1.77f, 47.99f, 0.38f, 0.25f},
                                {7.19f, 69.32f, 0.67f, 0.33f}};

// us of a launch in form f with `adapters` among the rows, or a negative number where it
// does not fit (a stage of 128 bytes a row, 256 where the adapters are not staged)
float form_cost(const Form& f, const FormCost& c, int64_t M, int64_t N, int64_t K, int elem, int r, int parts, int64_t adapters, int cus) {
  if (N % f.bn != 0 || K * elem % (f.staged ? 128 : 256) != 0) return -1.f;
  const int64_t tiles = (M + f.bm - 1) / f.bm * (N / f.bn);
  const int64_t per = (tiles + cus - 1) / cus, rounds = (per + f.occ - 1) / f.occ;
  const float k = c.s * (float)K / 1024.f;
  const float runs = fminf(fminf((float)f.bm, (float)M), 1.f + (float)(adapters - 1) * f.bm / M);
  const int steps = (r * parts + 15) / 16;
  return c.a + (float)(rounds - 1) * (c.a - 2.f) + (float)rounds * k + c.m * k * (float)(per - rounds) +
         c.e * runs * (float)steps * (float)per;
}

// the cheapest form, -1: none
int product_form(int dtype, int64_t M, int64_t N, int64_t K, int r, int parts, int64_t adapters, int cus) {
  int form = -1;
  float cost = 0.f;
  const FormCost* const costs = dtype == PK_DTYPE_F32 ? kCost32 : dtype == PK_DTYPE_F16 ? kCostF16 : kCostBf16;
  const int elem = dtype == PK_DTYPE_F32 ? 4 : 2;
  const int built = dtype == PK_DTYPE_F32 ? sizeof(kCost32) / sizeof(kCost32[0]) : sizeof(kForms) / sizeof(kForms[0]);
  for (int i = 0; i < built; ++i) {
    const float c = form_cost(kForms[i], costs[i], M, N, K, elem, r, parts, adapters, cus);
    if (c >= 0.f && (form < 0 || c < cost)) {
      form = i;
      cost = c;
    }
  }
  return form;
}

template <typename ST, int SILU>
int launch_product(const AdK<ST>& k, int64_t adapters, int cus, hipStream_t s) {
  constexpr int dtype = sizeof(ST) == 4 ? PK_DTYPE_F32 : __is_same(ST, bf16_t) ? PK_DTYPE_BF16 : PK_DTYPE_F16;
  switch (product_form(dtype, k.M, k.N, k.K, k.r, k.parts, adapters, cus)) {
    case 0: return launch_tile<ST, 16, 16, 1, 1, 4, 128, 4, SILU>(k, s);
    case 1: return launch_tile<ST, 16, 32, 1, 1, 4, 128, 4, SILU>(k, s);
    case 2: return launch_tile<ST, 32, 32, 1, 1, 4, 128, 4, SILU>(k, s);
    case 3: return launch_tile<ST, 32, 64, 1, 2, 4, 128, 3, SILU>(k, s);
    case 4: return launch_tile<ST, 64, 64, 2, 2, 2, 64, 4, SILU>(k, s);
    case 5: return launch_tile<ST, 64, 128, 2, 4, 1, 64, 3, SILU>(k, s);
    case 6: return launch_tile<ST, 128, 128, 2, 2, 1, 64, 2, SILU>(k, s);
    case 7:
      if constexpr (sizeof(ST) == 2) return launch_tile<ST, 256, 256, 2, 4, 1, 64, 2, SILU>(k, s);
    default:
      return fail(PK_ERR_UNSUPPORTED, "pk_adapter_linear: no form for %d -> %d", k.K, k.N);
  }
}

template <typename ST, int RW, int RT, int BN, int WN, int WK, int BKB, int S, int SILU>
int launch_few_t(AdK<ST> k, hipStream_t s) {
  k.mtiles = (k.M + 15) / 16;
  const int nt = k.N / BN;
  k.xm = xcd_split(k.mtiles, nt, 16, BN);
  dim3 grid((unsigned)(k.mtiles * nt));
  if (k.xm > 0) grid = dim3(8u, (unsigned)(k.mtiles / k.xm), (unsigned)(nt / (8 / k.xm)));
  hipLaunchKernelGGL((adapter_few_kernel<ST, RW, RT, BN, WN, WK, BKB, S, SILU>), grid, dim3(64 * WN * WK), 0, s, k);
  return check_launch("pk_adapter_linear");
}

template <typename ST, int RW, int RT, int SILU>
int launch_few_n(const AdK<ST>& k, int bn, hipStream_t s) {
  if (bn == 16) return launch_few_t<ST, RW, RT, 16, 1, 8, 1024, 2, SILU>(k, s);
  if (bn == 32) return launch_few_t<ST, RW, RT, 32, 1, 8, 1024, 2, SILU>(k, s);
  if (bn == 64) return launch_few_t<ST, RW, RT, 64, 2, 4, 256, 3, SILU>(k, s);
  return launch_few_t<ST, RW, RT, 128, 4, 2, 256, 3, SILU>(k, s);
}

template <typename ST, int SILU>
int launch_few(const AdK<ST>& k, int bn, hipStream_t s) {
  const bool wide = k.K * (int)sizeof(ST) == 2048;
  if (k.r <= 16) return wide ? launch_few_n<ST, 2048, 1, SILU>(k, bn, s) : launch_few_n<ST, 1024, 1, SILU>(k, bn, s);
  return wide ? launch_few_n<ST, 2048, 2, SILU>(k, bn, s) : launch_few_n<ST, 1024, 2, SILU>(k, bn, s);
}

// adapters that the rows of a plan with so many tiles have at most
int64_t most_adapters(int64_t rows, int64_t max_tiles) { return max_tiles - rows / kLowRows > 1 ? max_tiles - rows / kLowRows : 1; }

// Outputs a workgroup of the few-row form: the fewest that give no CU a second tile; 0
// where two launches are as fast.  The line is what a tile's adapters (as many as the
// plan may have) take of A, 96 KB.  In a graph, few-row form and two launches, 128 rows 512 ->
// 2048 bf16: rank 16, one adapter (16 KB) 7.8 us and 10.0, 3 a tile (46 KB) 9.0 and 10.4, 5 (78
// KB) 12.8 and 10.7, rank 32, 3 a tile (93 KB) 11.7 and 10.9; called one by one the second
// launch is 3.3 us of the host's besides.
int few_form(int64_t M, int64_t N, int64_t row_bytes, int r, int64_t adapters, int cus) {
  if ((row_bytes != 1024 && row_bytes != 2048) || r > 32) return 0;
  const float runs = fminf(fminf(16.f, (float)M), 1.f + (float)(adapters - 1) * 16.f / M);
  if (runs * (float)r * (float)row_bytes > 96.f * 1024.f) return 0;
  for (int bn = 16; bn <= 128; bn *= 2)
    if (N % bn == 0 && (M + 15) / 16 * (N / bn) <= cus) return bn;
  return 0;
}

// below 2^31 bytes: 32-bit offsets, and kNowhere past them
bool rows_ok(int64_t rows, int64_t stride, int64_t width, int bytes) {
  if (rows > 1 && (stride < width || stride >= (int64_t{1} << 31))) return false;
  return stride >= 0 && stride % (16 / bytes) == 0 &&
         ((rows - 1) * stride + width) * bytes < (int64_t{1} << 31);
}

template <typename ST>
int adapter_typed(const pk_adapter_linear_args* a, hipStream_t s) {
  const char* what = "pk_adapter_linear";
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
  const int few = few_form(a->rows, a->n, (int64_t)a->k * sizeof(ST), a->rank, most_adapters(a->rows, a->max_tiles), cu_count());
  const void* ptrs[9] = {a->x,     a->a,   a->b, a->weight, a->bias ? a->bias : a->x,
                         a->tiles, a->out, few ? a->x : a->workspace, a->scale};
  for (const void* q : ptrs) {
    if (!q) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
    if (q != a->scale && !aligned16(q)) return fail(PK_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  }
  if (!a->order || !a->ids) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  constexpr int E = sizeof(ST);
  const int parts = k_parts(a->max_tiles, a->rank, a->k);
  if (!rows_ok(a->rows, a->x_stride, a->k, E) || !rows_ok(a->n, a->weight_stride, a->k, E) ||
      !rows_ok(a->rows, a->out_stride, a->n, E) || !rows_ok(a->rows, low_row<ST>(a->rank, parts) / 4, low_row<ST>(a->rank, parts) / 4, 4) ||
      !rows_ok(a->rank, a->k, a->k, E) || !rows_ok(a->n, a->rank, a->rank, E))
    return fail(PK_ERR_INVALID, "%s: row strides must be multiples of 16 bytes, at least the row, and a tensor below 2^31 bytes", what);
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
  k.parts = parts;
  k.kpart = ((k.K / 64 + k.parts - 1) / k.parts) * 64;
  k.units = parts * low_blocks(k.r);
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const int64_t adapters = most_adapters(k.M, a->max_tiles);
  const int cus = cu_count();
  if (few) return a->activation == PK_ACT_SILU ? launch_few<ST, 1>(k, few, s) : launch_few<ST, 0>(k, few, s);
  if (a->max_tiles > 0) {
    const int rc = launch_low(k, a->max_tiles, s);
    if (rc != PK_OK) return rc;
  }
  return a->activation == PK_ACT_SILU ? launch_product<ST, 1>(k, adapters, cus, s) : launch_product<ST, 0>(k, adapters, cus, s);
}

}  // namespace
}  // namespace pk

extern "C" int64_t pk_adapter_workspace_bytes(int32_t dtype, int32_t rows, int32_t n, int32_t k, int32_t rank, int32_t max_tiles) {
  if (rows <= 0 || n <= 0 || rank <= 0 || k <= 0 || max_tiles < 0) return 0;
  const int64_t row = (int64_t)k * (dtype == PK_DTYPE_F32 ? 4 : 2);
  if (pk::few_form(rows, n, row, rank, pk::most_adapters(rows, max_tiles), pk::cu_count())) return 0;
  const int parts = pk::k_parts(max_tiles, rank, k);
  return rows * (int64_t)(dtype == PK_DTYPE_F16 ? pk::low_row<_Float16>(rank, parts) : pk::low_row<float>(rank, parts));
}

extern "C" int pk_adapter_linear_form(int32_t dtype, int32_t rows, int32_t n, int32_t k, int32_t rank, int32_t max_tiles, int32_t cus,
                                      pk_adapter_form* form) {
  pk::clear_error();
  if (!form || rows <= 0 || n <= 0 || n % 64 != 0 || k <= 0 || k % 64 != 0 || rank <= 0 || max_tiles < 0)
    return pk::fail(PK_ERR_INVALID, "pk_adapter_linear_form: need form, rows, rank > 0, max_tiles >= 0 and widths of multiples of 64");
  if (cus <= 0) cus = pk::cu_count();
  const int elem = dtype == PK_DTYPE_F32 ? 4 : 2;
  const int64_t adapters = pk::most_adapters(rows, max_tiles);
  const int few = pk::few_form(rows, n, (int64_t)k * elem, rank, adapters, cus);
  form->parts = few ? 1 : pk::k_parts(max_tiles, rank, k);
  const int i = few ? -1 : pk::product_form(dtype, rows, n, k, rank, form->parts, adapters, cus);
  if (!few && i < 0) return pk::fail(PK_ERR_UNSUPPORTED, "pk_adapter_linear_form: no form for %d -> %d", k, n);
  form->launches = few ? 1 : 2;
  form->tile_rows = few ? 16 : pk::kForms[i].bm;
  form->tile_columns = few ? few : pk::kForms[i].bn;
  return PK_OK;
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
