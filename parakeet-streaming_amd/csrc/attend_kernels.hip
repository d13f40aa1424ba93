// gfx950 attention of a text decoder: new tokens over a paged cache, and over the encoder's
// states; the norms and rotation of new queries and keys with their way into the pages.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "pk_common.h"
#include "pk_device.h"
#include "pk_scan.h"
#include "pk_tile.h"

namespace pk {

// ---------------------------------------------------------------------------
// head norms, rotation, append
//
// Bound by memory: a token's heads are read and written once. A workgroup takes kTok tokens:
// its threads first ask for their columns, then make the tokens' cosines and sines (one pair
// a frequency, shared by all heads) in LDS. A head is HD / VEC neighbouring lanes; its sum of
// squares is one DPP reduction, and the partner columns of a rotation are in lane l ^ span.

template <typename ST>
struct NormK {
  const ST* q;
  const ST* k;
  const ST* v;
  ST* out;
  ST* kp;  // the layer's slabs
  ST* vp;
  const ST* qw;  // or nullptr
  const ST* kw;
  const double* inv;
  const int32_t* pos;  // or nullptr: rows[b][0] + t
  const int32_t* rows;
  const int32_t* map;
  int64_t q_sb, q_st, k_sb, k_st, v_sb, v_st, o_sb, o_st, pos_sb, map_sb, rows_stride;
  int32_t B, T, Hq, Hkv, rotary, interleaved, page_shift;
  uint32_t places;  // num_pages * page_size
  float eps;
};

// cos and sin of position * inv_freq: the angle in turns in 64 bits, where its whole part
// goes, the rest in 32
__device__ static inline float2 turn_of(int32_t pos, double inv) {
  const double turns = (double)pos * (inv * 0.15915494309189535);  // 1 / 2 pi
  const float part = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.f * part, &s, &c);
  return float2{c, s};
}

// x of lane ^ SPAN
template <int SPAN>
__device__ static inline float of_partner(float x) {
  if constexpr (SPAN == 1) return dpp_f<0xB1>(x);                // quad_perm [1, 0, 3, 2]
  if constexpr (SPAN == 2) return dpp_f<0x4E>(x);                // quad_perm [2, 3, 0, 1]
  if constexpr (SPAN == 4) return dpp_f<0x1B>(dpp_f<0x141>(x));  // row_half_mirror: lane ^ 7, quad_perm [3, 2, 1, 0]: lane ^ 3
  if constexpr (SPAN == 8) return dpp_f<0x128>(x);               // row_ror 8
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(threadIdx.x & 16 ? r[0] : r[1]);
}

// A wave takes the 64 / LPH heads of an item at once (q's, k's and v's in a row, so that an item is 1 KB), TOK tokens'
// items over the workgroup's waves; U items' loads are on their way together. 15.6 K tokens of 16 + 2 + 2
// heads of 128 in bf16, half of them with a place, 144 MB read and written: 28.6 us, 5.0 TB/s (a large copy: 5.2). Of so many tokens the
// caches keep nothing, so their stores go past them: 33.6 us through them; loads past them as well 33.7.
template <typename ST, int HD, int TOK, int U>
__global__ void __launch_bounds__(256) qk_norm_append_kernel(const NormK<ST> p) {
  constexpr int VEC = Tr<ST>::VEC, LPH = HD / VEC, CB = 64 / (int)sizeof(ST), HPI = 64 / LPH;
  __shared__ __align__(16) float2 cs[TOK][HD];  // of a column: the cosine, and the sine with the sign that its partner has in it
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int heads = p.Hq + 2 * p.Hkv, per = (heads + HPI - 1) / HPI, half = p.rotary >> 1;
  const uint32_t total = (uint32_t)p.B * (uint32_t)p.T, first = blockIdx.x * (uint32_t)TOK;  // below 2^31
  const int tokens = (int)min((uint32_t)TOK, total - first), items = tokens * per;
  const int c = (lane & (LPH - 1)) * VEC;

  u32x4 raw[U];
  ST* to[U];
  // asks for item `item`: its token's row, and where it goes (nullptr: nowhere)
  auto ask = [&](int u, int item) {
    to[u] = nullptr;
    if (item >= items) return;
    const int t = item / per, head0 = (item - t * per) * HPI;
    const uint32_t row = first + t, b = row / (uint32_t)p.T, at = row - b * (uint32_t)p.T;
    if (head0 + HPI <= p.Hq) {  // wave-uniform: queries alone, by their lanes' bytes from a place that all share
      const int col = head0 * HD;
      raw[u] = ld16(p.q + b * p.q_sb + at * p.q_st + col + (uint32_t)(lane * VEC));
      to[u] = p.out + b * p.o_sb + at * p.o_st + col + (uint32_t)(lane * VEC);
      return;
    }
    const int head = head0 + lane / LPH;
    const uint32_t place = (uint32_t)p.map[b * p.map_sb + at];
    const ST* from = nullptr;
    if (head < p.Hq) {
      const int col = head * HD + c;
      from = p.q + b * p.q_sb + at * p.q_st + col;
      to[u] = p.out + b * p.o_sb + at * p.o_st + col;
    } else if (head < heads && place < p.places) {
      const bool key = head < p.Hq + p.Hkv;
      const int col = (head - p.Hq - (key ? 0 : p.Hkv)) * HD + c, rest = (int)place & ((1 << p.page_shift) - 1);
      from = key ? p.k + b * p.k_sb + at * p.k_st + col : p.v + b * p.v_sb + at * p.v_st + col;
      to[u] = (key ? p.kp : p.vp) + (int64_t)(place >> p.page_shift) * (((int64_t)p.Hkv * HD) << p.page_shift) +
              ((int64_t)(col / CB) * CB << p.page_shift) + (int64_t)rest * CB + col % CB;
    }
    raw[u] = to[u] ? ld16(from) : u32x4{0u, 0u, 0u, 0u};
  };
#pragma unroll
  for (int u = 0; u < U; ++u) ask(u, wave + 4 * u);
  float qg[VEC], kg[VEC];
  if (p.qw) Tr<ST>::unpack(ld16(p.qw + c), qg);
  if (p.kw) Tr<ST>::unpack(ld16(p.kw + c), kg);
  for (int i = threadIdx.x; i < tokens * half; i += 256) {
    const int t = i / half, f = i - t * half;
    const uint32_t row = first + t, b = row / (uint32_t)p.T, at = row - b * (uint32_t)p.T;
    const float2 x = turn_of(p.pos ? p.pos[b * p.pos_sb + at] : p.rows[b * p.rows_stride] + (int32_t)at, p.inv[f]);
    cs[t][p.interleaved ? 2 * f : f] = float2{x.x, -x.y};
    cs[t][p.interleaved ? 2 * f + 1 : half + f] = x;
  }
  __syncthreads();
  // the columns of an item in registers: norm, rotation with the partners `span` lanes away (0: beside it)
  auto turn = [&](float (&x)[VEC], const float2* f, bool turned, auto span) {
    constexpr int SPAN = decltype(span)::value;
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float other = SPAN == 0 ? x[e ^ 1] : of_partner<SPAN>(x[e]);
      y[e] = fmaf(other, f[e].y, x[e] * f[e].x);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = turned ? y[e] : x[e];
  };
  auto make = [&](int u, int item, auto mixed) {
    constexpr bool MIXED = decltype(mixed)::value;  // keys or values among the item's heads
    const int t = item / per, head = (item - t * per) * HPI + lane / LPH;
    const bool key = MIXED && head >= p.Hq, value = MIXED && head >= p.Hq + p.Hkv;
    float x[VEC];
    Tr<ST>::unpack(raw[u], x);
    if (key ? p.kw != nullptr : p.qw != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss = fmaf(x[e], x[e], ss);
      ss = group_sum<LPH>(ss);
      const float r = __builtin_amdgcn_rsqf(ss * (1.f / HD) + p.eps);  // 1 ulp
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] *= r * (key ? kg[e] : qg[e]);
    }
    if (half > 0) {
      const bool turned = !value && c < p.rotary;
      const float2* const f = &cs[t][c < p.rotary ? c : 0];
      const int span = half / VEC;
      using std::integral_constant;
      if (p.interleaved)
        turn(x, f, turned, integral_constant<int, 0>());
      else if (span == LPH / 2)
        turn(x, f, turned, integral_constant<int, LPH / 2>());
      else if (span == LPH / 4)
        turn(x, f, turned, integral_constant<int, LPH / 4>());
      else if (span == 4)
        turn(x, f, turned, integral_constant<int, 4>());
      else if (span == 2)
        turn(x, f, turned, integral_constant<int, 2>());
      else
        turn(x, f, turned, integral_constant<int, 1>());
    }
    const u32x4 made = value ? raw[u] : Tr<ST>::pack(x);
    if (!to[u]) return;
    if constexpr (TOK == 8)
      __builtin_nontemporal_store(made, reinterpret_cast<u32x4*>(to[u]));
    else
      st16(to[u], made);
  };
  for (int i0 = wave; i0 < items; i0 += 4 * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int item = i0 + 4 * u;
      if (item >= items) break;  // wave-uniform
      if ((item % per + 1) * HPI <= p.Hq)
        make(u, item, std::false_type());
      else
        make(u, item, std::true_type());
    }
#pragma unroll
    for (int u = 0; u < U; ++u) ask(u, i0 + 4 * (U + u));
  }
}

// ---------------------------------------------------------------------------
// attention
//
// out_i = sum_j softmax_j(scale q_i . k_j) v_j.  Rows are (token, query head of a key head)
// pairs; where keys are differs (pages, or a tensor of states), what is done with them does not.

template <typename ST>
struct AttendK {
  const ST* q;
  ST* out;
  const unsigned char* k;  // the layer's slab, or the states
  const unsigned char* v;
  int64_t q_sb, q_st, o_sb, o_st;    // elements
  int64_t k_sb, k_st, v_sb, v_st;    // states: bytes
  const int32_t* rows;               // pages
  int64_t rows_stride, page_bytes;
  int32_t max_pages, page_shift, num_pages;
  const int32_t* lengths;
  int32_t B, T, Hq, Hkv, G, left, states;
  float scale;  // times log2(e)
  int32_t R;                 // rows of a key head: T * G
  int32_t row_tiles, splits;  // workgroups along the rows, and along the keys
  int32_t order, key_bits;    // Order; bits of the most keys
  float* part;   // splits > 1: [B * Hkv * R][splits][HD] sums over a split's keys
  float2* ml;    // and [B * Hkv * R][splits] their {maximum in log2 units, sum of weights}
};

// Streams in the order of the batch; the longest first, 256 at a time; so, but every second one from the end
enum Order { kAsTheyAre, kLongFirst, kFolded };

// A row's maximum before it has met a key; and of one that has met keys whose scores were all -inf, since a softmax
// of them is NaN where one of no keys is zeros here.
constexpr float kNone = -__builtin_inff(), kLeast = -__FLT_MAX__;
// 1 / l, of a row of sum l and maximum m
__device__ static inline float quotient(float m, float l) { return l != 0.f ? 1.f / l : m == kNone ? 0.f : __builtin_nanf(""); }

// Weights are 2^(score - m), m following the maximum. fp16 loses bits of those below 2^-14 and all of those below
// 2^-25, and a long tail of them can be a good part of the sum; it ends at 2^16 only, so there m stays below the maximum, by
// what keeps the largest weights at 2^kTop. The quotient cancels it.
template <typename ST>
constexpr float kTop = __is_same(ST, _Float16) ? 15.f : 0.f;

// fp32's steps reach 1/2 at kFar: past it 2^(a score's exact product with the scale - a rounded maximum) may be anything, up to
// infinity. Rows with such maxima are made again from scores that are rounded as their maximum is (attend_row), by parts
// whose sum is NaN.
constexpr float kFar = 4194304.f;
__device__ static inline float2 part_of(float m, float l) { return float2{m, m != kNone && fabsf(m) >= kFar ? __builtin_nanf("") : l}; }
__device__ static inline float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// what a workgroup needs of a stream
struct StreamOf {
  int32_t A;     // position of token 0 (pages)
  int32_t n;     // tokens
  int32_t end;   // keys
};

template <typename ST, bool PAGED>
__device__ static inline StreamOf stream_of(const AttendK<ST>& p, int b) {
  StreamOf s;
  if constexpr (PAGED) {
    s.n = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
    s.A = min(max(p.rows[b * p.rows_stride], 0), 0x7fffffff - p.T);
    s.end = s.A + s.n;
  } else {
    s.n = p.T;
    s.A = 0;
    s.end = p.lengths ? min(max(p.lengths[b], 0), p.states) : p.states;
  }
  return s;
}

// keys that token i sees: [first, last]
template <typename ST, bool PAGED>
__device__ static inline int2 seen_by(const AttendK<ST>& p, const StreamOf& s, int i) {
  if constexpr (PAGED) return int2{max(0, s.A + i - p.left), s.A + i};
  return int2{0, s.end - 1};
}

// Byte offset, in the slab or the states, of key j's first column of key head h; -1: not there.
// Its next 64 bytes are block_step further (pages hold column blocks).
template <typename ST, bool PAGED>
__device__ static inline int64_t key_at(const AttendK<ST>& p, int b, int hd_bytes, int h, int j, bool v) {
  if constexpr (PAGED) {
    const int32_t page = p.rows[b * p.rows_stride + 1 + ((uint32_t)j >> p.page_shift) % (uint32_t)p.max_pages];
    if ((uint32_t)page >= (uint32_t)p.num_pages) return -1;
    return page * p.page_bytes + ((int64_t)(h * hd_bytes) << p.page_shift) + (((uint32_t)j & ((1u << p.page_shift) - 1u)) << 6);
  }
  return b * (v ? p.v_sb : p.k_sb) + j * (v ? p.v_st : p.k_st) + (int64_t)h * hd_bytes;
}

// One row by one wave, without the matrix cores: 64 keys at a time, a key a lane for the
// scores, columns over the lanes for the sums. q: the row, in fp32, in LDS. Keys first ..
// first + n - 1 (counted: positions run up to 2^31 - 1). Gives the
// maximum (log2 units), the sum, and the sums of columns lane + 64 c.
template <typename ST, int HD, bool PAGED>
__device__ static inline void attend_row(const AttendK<ST>& p, int b, int h, const float* q, int first, int n, float& m, float& l,
                                         float (&acc)[HD / 64]) {
  constexpr int VEC = Tr<ST>::VEC, CB = 64 / (int)sizeof(ST), E = (int)sizeof(ST);
  const int lane = threadIdx.x & 63;
  const int64_t step = PAGED ? (int64_t)64 << p.page_shift : 64;
  m = kNone;
  l = 0.f;
  bool met = false;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) acc[c] = 0.f;
  for (int d0 = 0; d0 < n; d0 += 64) {
    const int64_t at = d0 + lane < n ? key_at<ST, PAGED>(p, b, HD * E, h, first + d0 + lane, false) : -1;
    const int64_t vat = PAGED || at < 0 ? at : key_at<ST, PAGED>(p, b, HD * E, h, first + d0 + lane, true);
    met = met || __any(at >= 0);
    float s = kNone;
    if (at >= 0) {
      float d = 0.f;
      for (int c = 0; c < HD; c += VEC) {
        float x[VEC];
        Tr<ST>::unpack(*reinterpret_cast<const u32x4*>(p.k + at + c / CB * step + c % CB * E), x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) d = fmaf(x[e], q[c + e], d);
      }
      s = rounded_product(d, p.scale);
    }
    float top = s;
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    bool nan = __any(s != s);
    const float now = fmaxf(m, top);
    const float keep = now == kNone ? 1.f : __builtin_amdgcn_exp2f(m - now);
    const float e = at < 0 || now == kNone ? 0.f : __builtin_amdgcn_exp2f(s - now);
    float sum = group_sum<64>(e);
    if (nan) sum = __builtin_nanf("");
    l = l * keep + sum;
    m = now;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) acc[c] *= keep;
    if (l != l) {  // whatever follows
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) acc[c] = l;
      break;
    }
    // eight keys' values on their way at a time; of one that is not there, place 0's, which are not used
    bool gone = true;
    for (int u0 = 0; u0 < min(64, n - d0); u0 += 8) {
      float x[8][HD / 64], w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int lo = __builtin_amdgcn_readlane((int)vat, u0 + u), hi = __builtin_amdgcn_readlane((int)(vat >> 32), u0 + u);
        const int64_t va = (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
        w[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), u0 + u));
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) {
          const int col = lane + 64 * c;
          const float y = from_st(*reinterpret_cast<const ST*>(p.v + max(va, (int64_t)0) + col / CB * step + col % CB * E));
          x[u][c] = va < 0 ? 0.f : y;
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) acc[c] = fmaf(w[u], x[u][c], acc[c]);
    }
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) gone = gone && acc[c] != acc[c];
    if (__all(gone)) break;
  }
  if (met) m = fmaxf(m, kLeast);
}

// ---- few rows

// matrix products of 64 bytes of columns (a column block): D[a's row][b's row] += a . b, where
// lane (r = lane & 15, g = lane >> 4) holds bytes 16 g .. 16 g + 15 of row r of each, and gets D of
// rows 4 g .. 4 g + 3 of a with row r of b. fp32: element e of a lane is column 4 g + e, so
// step e multiplies columns e, 4 + e, 8 + e and 12 + e.
template <typename ST>
__device__ static inline f32x4_t mma_block(const u32x4 a, const u32x4 b, f32x4_t c) {
  if constexpr (sizeof(ST) == 2) {
    return MmaL<ST>::k32(a, b, c);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
}

// largest of the four lanes l & 15, l & 15 + 16, ...
__device__ static inline float max_of_groups(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ static inline float sum_of_groups(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// what a workgroup works on
struct ItemOf {
  int32_t b, hk, row0, split;
  bool live;
};

// Workgroup -> (stream and key head and split, row tile): workgroups go to the XCDs in turn, and
// the row tiles of the same keys to the same one, whose L2 then has them. Streams of different lengths: the
// longest first, so that the last workgroups to end are short ones; where all are on the GPU at once,
// and none waits for another, every second one in the other order, so that a CU has a long and a short one
// (60 x 4 rows over up to 1500 states: 54.7 us as they are, 43.3 folded; 8 x 197 rows in fp32 over up to
// 751: 31.8 and 25.4; 100 streams of 8 heads of 64 over up to 3000 tokens, longest first: 62.0 and 57.3).
template <typename ST, bool PAGED>
__device__ static inline ItemOf item_of(const AttendK<ST>& p, int rows, StreamOf& s) {
  const uint32_t x = blockIdx.x & 7, y = blockIdx.x >> 3;
  const uint32_t tile = y % (uint32_t)p.row_tiles, u = y / (uint32_t)p.row_tiles * 8 + x;
  const uint32_t unit = u / (uint32_t)p.splits;
  ItemOf it;
  it.split = (int32_t)(u - unit * (uint32_t)p.splits);
  it.b = (int32_t)(unit / (uint32_t)p.Hkv);
  it.hk = (int32_t)(unit - (uint32_t)it.b * (uint32_t)p.Hkv);
  it.row0 = (int32_t)tile * rows;
  it.live = it.b < p.B;
  if (!it.live) return it;
  if (p.order == kAsTheyAre) {
    s = stream_of<ST, PAGED>(p, it.b);
    return it;
  }
  // the stream that has `want` longer ones before it, of the 256 around b, four a lane; by the six highest bits of the
  // keys that it has
  constexpr int N = 4;
  const int lane = threadIdx.x & 63, b0 = it.b & -(64 * N), n = min(64 * N, p.B - b0);
  StreamOf mine[N];
  uint32_t keys[N];
  uint64_t left[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    keys[j] = 0;
    left[j] = 0;
    if (64 * j >= n) continue;
    mine[j] = stream_of<ST, PAGED>(p, b0 + min(64 * j + lane, n - 1));
    keys[j] = (uint32_t)(PAGED ? (mine[j].n > 0 ? min(mine[j].A, p.left) + mine[j].n : 0) : mine[j].end);
    left[j] = n >= 64 * (j + 1) ? ~0ull : (1ull << (n - 64 * j)) - 1;
  }
  int want = it.b - b0;
  if (p.order == kFolded) {  // the second half of the 256, or of the batch's, from the end
    const bool one = p.B <= 64 * N;
    const int half = one ? (n + 1) >> 1 : 0;
    if (one ? want >= half : 2 * (b0 / (64 * N)) >= (p.B + 64 * N - 1) / (64 * N)) want = n - 1 - (want - half);
  }
  for (int bit = p.key_bits - 1, last = max(p.key_bits - 6, 0); bit >= last; --bit) {
    uint64_t longer[N];
    int c = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (64 * j >= n) continue;
      longer[j] = __ballot(keys[j] >> bit & 1) & left[j];
      c += __popcll(longer[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (64 * j < n) left[j] = want < c ? longer[j] : left[j] & ~longer[j];
    want -= want < c ? 0 : c;
  }
  // of those that are left, the want-th
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (64 * j >= n) continue;
    const int c = __popcll(left[j]);
    if (want >= 0 && want < c) {
      const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(left[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)left[j], 0));
      const int at = __builtin_ctzll(__ballot((left[j] >> lane & 1) && before == want));
      it.b = b0 + 64 * j + at;
      s.A = __builtin_amdgcn_readlane(mine[j].A, at);
      s.n = __builtin_amdgcn_readlane(mine[j].n, at);
      s.end = __builtin_amdgcn_readlane(mine[j].end, at);
    }
    want -= c;
  }
  return it;
}

// Keys of a row tile, in tiles of KT: number d of a key counts from k0 (a multiple of KT, so that
// a tile meets few pages); some row sees keys lo .. hi. The split has tiles t0 .. t1 - 1.
struct KeysOf {
  int32_t k0, lo, hi, t0, t1;
};

template <typename ST, bool PAGED, int KT>
__device__ static inline KeysOf keys_of(const AttendK<ST>& p, const StreamOf& s, int row0, int rows, int split) {
  const int i0 = row0 / p.G, i1 = min((min(row0 + rows, p.R) - 1) / p.G, s.n - 1);
  KeysOf k{0, 0, -1, 0, 0};
  if (i1 < i0) return k;
  const int first = seen_by<ST, PAGED>(p, s, i0).x, last = seen_by<ST, PAGED>(p, s, i1).y;
  if (last < first) return k;
  k.k0 = first & ~(KT - 1);
  k.lo = first - k.k0;
  k.hi = last - k.k0;
  // at least a tile a wave, so that short streams of a long batch leave splits empty
  const int tiles = k.hi / KT + 1, per = max((tiles + p.splits - 1) / p.splits, 4);
  k.t0 = min(split * per, tiles);
  k.t1 = min(k.t0 + per, tiles);
  return k;
}

// Whether a row that sees keys lo .. hi and whose maximum is none all the same has met a key in its split: the scores were
// -inf then. Rare, so it is looked up when all is done.
template <typename ST, bool PAGED, int KT>
__device__ static inline bool has_met(const AttendK<ST>& p, int b, const KeysOf& keys, int lo, int hi, bool none) {
  const int from = max(lo, keys.t0 * KT), to = min(hi, keys.t1 * KT - 1);
  const bool met = none && from <= to;
  if constexpr (!PAGED) return met;
  if (!__any(met)) return false;
  // of the pages that the split meets, whether there is one with a key of the row
  const int32_t* const ring = p.rows + b * p.rows_stride + 1;
  auto page_of = [&](int d) { return (int)(((uint32_t)keys.k0 + (uint32_t)d) >> p.page_shift); };
  const int page0 = page_of(max(keys.lo, keys.t0 * KT)), pages = page_of(min(keys.hi, keys.t1 * KT - 1)) - page0 + 1;
  uint64_t any = 0;
  for (int i0 = 0; i0 < pages; i0 += 64) {
    const int i = min(i0 + (int)(threadIdx.x & 63), pages - 1);
    const uint64_t there = __ballot((uint32_t)ring[(uint32_t)(page0 + i) % (uint32_t)p.max_pages] < (uint32_t)p.num_pages);
    const int x = max(page_of(from) - page0 - i0, 0), y = min(page_of(to) - page0 - i0, 63);
    any |= x <= y ? there >> x & (~0ull >> (63 - (y - x))) : 0ull;
  }
  return met && any != 0;
}

// The end of a workgroup's rows: sums over the waves' parts of the keys (in LDS, scaled to their largest
// maximum; ml: each part's own maximum and sum of weights), the quotient, or the split's part.
// WAVES parts of [rows][HD + 4] floats at `sums`.
template <typename ST, int HD, bool PAGED, int ROWS, int WAVES, int THREADS, int KT>
__device__ static inline void attend_end(const AttendK<ST>& p, const ItemOf& it, const StreamOf& s, const KeysOf& keys, const float* sums,
                                         const float2* ml, float* qs) {
  constexpr int VEC = 8, PER = HD / VEC, STRIDE = HD + 4, N = (ROWS * PER + THREADS - 1) / THREADS;
  static_assert(ROWS * PER % 64 == 0, "a wave has rows in all lanes or in none");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  constexpr uint64_t kRow = (1ull << PER) - 1;  // a row is PER neighbouring lanes
  float o[N][VEC], m[N], l[N];
  uint64_t bad[N];
#pragma unroll
  for (int y = 0; y < N; ++y) {
    const int x = y * THREADS + threadIdx.x, r = x / PER, c = (x - r * PER) * VEC;
    bad[y] = 0;
    if (r >= ROWS) continue;
    m[y] = kNone;
    l[y] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m[y] = fmaxf(m[y], ml[w * ROWS + r].x);
    const float base = m[y] == kNone ? 0.f : m[y];
    if (__builtin_expect(keys.t0 < keys.t1 && __any(m[y] == kNone && it.row0 + r < p.R), 0)) {
      const int i = min(it.row0 + r, p.R - 1) / p.G;
      const int2 seen = seen_by<ST, PAGED>(p, s, i);
      const bool none = m[y] == kNone && it.row0 + r < p.R && i < s.n;
      if (has_met<ST, PAGED, KT>(p, it.b, keys, seen.x - keys.k0, seen.y - keys.k0, none)) m[y] = kLeast;
    }
#pragma unroll
    for (int w = 0; w < WAVES; ++w) l[y] = fmaf(ml[w * ROWS + r].y, __builtin_amdgcn_exp2f(ml[w * ROWS + r].x - base), l[y]);
    float t = l[y];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      o[y][e] = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) o[y][e] += sums[(w * ROWS + r) * STRIDE + c + e];
      t = fmaf(o[y][e], 0.f, t);
    }
    bad[y] = __ballot(it.row0 + r < p.R && !(fabsf(t) < __builtin_inff()));
  }
#pragma unroll
  for (int y = 0; y < N; ++y) {
    const int x = y * THREADS + threadIdx.x, r = x / PER, c = (x - r * PER) * VEC, row = it.row0 + r;
    if (r >= ROWS || row >= p.R) continue;
    if (bad[y] >> (lane & -PER) & kRow) continue;
    const int i = row / p.G, h = it.hk * p.G + row - i * p.G;
    if (p.splits > 1) {
      const int64_t at = (((int64_t)it.b * p.Hkv + it.hk) * p.R + row) * p.splits + it.split;
      float* const to = p.part + at * HD + c;
      *reinterpret_cast<f32x4_t*>(to) = f32x4_t{o[y][0], o[y][1], o[y][2], o[y][3]};
      *reinterpret_cast<f32x4_t*>(to + 4) = f32x4_t{o[y][4], o[y][5], o[y][6], o[y][7]};
      if (c == 0) p.ml[at] = float2{m[y], l[y]};
    } else {
      const float inv = quotient(m[y], l[y]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[y][e] *= inv;
      ST* const to = p.out + it.b * p.o_sb + i * p.o_st + (int64_t)h * HD + c;
      st16(to, Tr<ST>::pack(o[y]));
      if constexpr (sizeof(ST) == 4) st16(to + 4, Tr<ST>::pack(o[y] + 4));
    }
  }
  // A row that is not finite may have met, as 0 times it, a value that it does not see, or scores past kFar: it is made again
  // from the keys that it sees, one by one (rare). It is not written yet: out may be the query that is read again.
  uint64_t some = bad[0];
#pragma unroll
  for (int y = 1; y < N; ++y) some |= bad[y];
  if (__builtin_expect(some == 0, 1)) return;
  for (int z = 0; z < N * (64 / PER); ++z) {
    uint64_t rows = bad[0];
#pragma unroll
    for (int y = 1; y < N; ++y) rows = z / (64 / PER) == y ? bad[y] : rows;
    if (rows == 0) {  // wave-uniform, as rows is: on to the next 64 / PER rows
      z |= 64 / PER - 1;
      continue;
    }
    if (!(rows >> (z % (64 / PER) * PER) & kRow)) continue;
    const int r = (z / (64 / PER) * THREADS + wave * 64) / PER + z % (64 / PER), row = it.row0 + r, i = row / p.G, h = it.hk * p.G + row % p.G;
    const ST* const q = p.q + it.b * p.q_sb + i * p.q_st + (int64_t)h * HD;
    for (int c = lane; c < HD; c += 64) qs[wave * HD + c] = from_st(q[c]);
    wave_lds_sync();
    const int2 seen = seen_by<ST, PAGED>(p, s, i);
    const int first = max(seen.x, keys.k0 + keys.t0 * KT);
    // a token past the stream's sees nothing
    const int n = i < s.n ? min(seen.y - keys.k0, keys.t1 * KT - 1) - (first - keys.k0) + 1 : 0;
    float m, l, acc[HD / 64];
    attend_row<ST, HD, PAGED>(p, it.b, it.hk, qs + wave * HD, first, n, m, l, acc);
    const float inv = quotient(m, l);
    const int64_t at = (((int64_t)it.b * p.Hkv + it.hk) * p.R + row) * p.splits + it.split;
    ST* const to = p.out + it.b * p.o_sb + i * p.o_st + (int64_t)h * HD;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      if (p.splits > 1)
        p.part[at * HD + lane + 64 * c] = acc[c];
      else
        to[lane + 64 * c] = to_st<ST>(l != 0.f ? acc[c] / l : inv);
    }
    if (p.splits > 1 && lane == 0) p.ml[at] = float2{m, l};
    wave_lds_sync();
  }
}

// Up to 16 RT rows of a key head a workgroup; its 4 waves take tiles of KT keys in turn. Bound by the
// reads of K and V, once (128 streams of up to 4096 tokens, 538 MB: 88 us, 6.1 TB/s; in fp32 by the matrix cores: 8 x 197
// rows of 8 heads of 64 over up to 751, 25 us), so a wave keeps a tile of both on its way: K's registers are
// asked for again when the scores are made, V's when they are staged, the page numbers a tile ahead.
// Products are taken transposed, keys (then columns of V) as rows: a lane has one query, 4 keys a
// register group, so maxima and sums are in the lane but for 4 lanes, and the weights are the next
// product's operand where they are. 16-bit types: two tiles of 16 keys make one step of 32, in
// the order that the registers have; V comes back transposed from LDS; weights go into the
// product as a high and a low 16-bit part, which costs nothing here and keeps 2^-16 or better of them (fp16: of those from
// 2^-24 of the largest on; the low part ends at 2^-40 of it).
// Where keys are: a tensor of states; pages of 16 frames and more, so that 16 keys from a multiple of 16 on are of
// one page, whose number is a scalar; smaller pages, looked up key by key.
// Pages that one row tile reads are read past the caches (128 streams of up to 4096, before they were put in order: 119 us cached, 107 so); rows of states
// are not, since a load has half of a 128-byte line of each (60 x 4 rows over up to 1500: 43 us, 63 past the caches).
enum Source { kStates, kPages, kSmallPages };
template <typename ST, int HD, Source SRC, int RT, bool STREAM>
__global__ void __launch_bounds__(256, 2) attend_few_kernel(const AttendK<ST> p) {
  constexpr bool PAGED = SRC != kStates;
  constexpr int NW = 4;
  constexpr int E = (int)sizeof(ST), ROWS = 16 * RT, SUB = E == 2 ? 2 : 1, KT = 16 * SUB, NB = HD * E / 64, NT = HD / 16;
  constexpr int VROW = HD * E + 16;  // bytes of a staged row of V: 16 more spread the rows over the banks
  constexpr int STRIDE = HD + 4;
  constexpr int kStage = NW * KT * VROW, kSums = NW * ROWS * STRIDE * 4;
  __shared__ __align__(16) unsigned char smem[kStage > kSums ? kStage : kSums];
  __shared__ float2 ml[NW * ROWS];
  __shared__ float qs[NW * HD];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  StreamOf s;
  const ItemOf it = item_of<ST, PAGED>(p, ROWS, s);
  if (!it.live) return;
  const KeysOf keys = keys_of<ST, PAGED, KT>(p, s, it.row0, ROWS, it.split);

  // the rows: their queries and what they see
  u32x4 q[RT][NB];
  int lo[RT], hi[RT], all_lo = 0, all_hi = 0x7fffffff;
  bool live[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = it.row0 + 16 * t + r16, i = min(row, p.R - 1) / p.G, gq = min(row, p.R - 1) - i * p.G;
    const ST* const from = p.q + it.b * p.q_sb + i * p.q_st + (int64_t)(it.hk * p.G + gq) * HD + g * (16 / E);
#pragma unroll
    for (int c = 0; c < NB; ++c) q[t][c] = ld16(from + c * (64 / E));
    // a row past the stream's tokens sees what its last token sees, and gives nothing in the end
    live[t] = i < s.n;
    const int2 seen = seen_by<ST, PAGED>(p, s, min(i, s.n - 1));
    lo[t] = seen.x - keys.k0;
    hi[t] = seen.y - keys.k0;
    all_lo = max(all_lo, lo[t]);
    all_hi = min(all_hi, hi[t]);
  }
  for (int d = 1; d < 16; d <<= 1) {
    all_lo = max(all_lo, __shfl_xor(all_lo, d));
    all_hi = min(all_hi, __shfl_xor(all_hi, d));
  }
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  f32x4_t o[RT][NT];
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = kNone;
    l[t] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) o[t][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  if (keys.t0 < keys.t1) {
    const int64_t step = PAGED ? (int64_t)64 << p.page_shift : 64;
    const unsigned char* const kb = p.k + (PAGED ? (int64_t)it.hk * (HD * E) << p.page_shift : it.b * p.k_sb + (int64_t)it.hk * (HD * E));
    const unsigned char* const vb = p.v + (PAGED ? (int64_t)it.hk * (HD * E) << p.page_shift : it.b * p.v_sb + (int64_t)it.hk * (HD * E));
    const int32_t* const ring = PAGED ? p.rows + it.b * p.rows_stride + 1 : nullptr;
    // The page numbers of tile t: of its 16 keys u, or of key lane % KT; -1 where no row of the workgroup
    // sees any. Read without a branch, so that the loads that go on are counted exactly.
    struct Pages {
      int32_t of[SUB];
    };
    auto pages_of = [&](int t) {
      Pages x{};
      if constexpr (SRC == kPages) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          const int d = t * KT + 16 * u;
          const bool in = t < keys.t1 && d + 15 >= keys.lo && d <= keys.hi;
          const uint32_t entry = (((uint32_t)keys.k0 + (uint32_t)(in ? d : keys.lo)) >> p.page_shift) % (uint32_t)p.max_pages;
          const int32_t page = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(ring))[__builtin_amdgcn_readfirstlane(entry)];
          x.of[u] = in ? page : -1;
        }
      } else if constexpr (SRC == kSmallPages) {
        const int d = t * KT + (lane & (KT - 1));
        const bool in = t < keys.t1 && d >= keys.lo && d <= keys.hi;
        const int32_t page = ring[(((uint32_t)keys.k0 + (uint32_t)(in ? d : keys.lo)) >> p.page_shift) % (uint32_t)p.max_pages];
        x.of[0] = in ? page : -1;
      }
      return x;
    };
    // Of 16 keys u of a tile: a place that all lanes share, a lane's bytes from there, and whether its key is there
    // (what memory holds for one that is not is not used).
    int64_t ks[SUB], vs[SUB];
    uint32_t kl[SUB], vl[SUB];
    bool ok[SUB];
    auto places = [&](int t, const Pages& pages) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int d0 = t * KT + 16 * u, d = d0 + r16;
        ok[u] = t < keys.t1 && d >= keys.lo && d <= keys.hi;
        if constexpr (SRC == kStates) {
          const int at = min(d0, keys.hi), more = min(r16, keys.hi - at);  // rows past the last are not touched
          ks[u] = at * p.k_st;
          vs[u] = at * p.v_st;
          kl[u] = (uint32_t)more * (uint32_t)p.k_st + g * 16;
          vl[u] = (uint32_t)more * (uint32_t)p.v_st + g * 16;
        } else if constexpr (SRC == kPages) {
          const bool there = (uint32_t)pages.of[u] < (uint32_t)p.num_pages;
          ok[u] = ok[u] && there;
          ks[u] = vs[u] = (there ? pages.of[u] : 0) * p.page_bytes + ((((uint32_t)keys.k0 + (uint32_t)d0) & ((1u << p.page_shift) - 1u)) << 6);
          kl[u] = vl[u] = r16 * 64 + g * 16;
        } else {
          const int32_t mine = __shfl(pages.of[0], 16 * u + r16);
          ok[u] = (uint32_t)mine < (uint32_t)p.num_pages;
          ks[u] = vs[u] = ok[u] ? mine * p.page_bytes + ((((uint32_t)keys.k0 + (uint32_t)d) & ((1u << p.page_shift) - 1u)) << 6) : 0;
          kl[u] = vl[u] = g * 16;
        }
      }
    };
    u32x4 kr[SUB][NB], vr[SUB][NB];
    auto ask = [&](u32x4 (&x)[SUB][NB], const unsigned char* base, const int64_t (&at)[SUB], const uint32_t (&off)[SUB]) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int c = 0; c < NB; ++c) {
          const u32x4* const from = reinterpret_cast<const u32x4*>(base + at[u] + c * step + off[u]);
          x[u][c] = STREAM ? __builtin_nontemporal_load(from) : *from;
        }
    };
    unsigned char* const stage = smem + wave * (KT * VROW);
    int t = keys.t0 + wave;
    places(t, pages_of(t));
    Pages next = pages_of(t + NW);  // ahead of the loads, as in the loop: waiting for it is no wait for them
    __builtin_amdgcn_sched_barrier(0);
    ask(kr, kb, ks, kl);
    __builtin_amdgcn_sched_barrier(0);
    ask(vr, vb, vs, vl);
    for (; t < keys.t1; t += NW) {
      bool now[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) now[u] = ok[u];
      f32x4_t x[RT][SUB];
#pragma unroll
      for (int a = 0; a < RT; ++a)
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          x[a][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < NB; ++c) x[a][u] = mma_block<ST>(kr[u][c], q[a][c], x[a][u]);
        }
      __builtin_amdgcn_sched_barrier(0);
      places(t + NW, next);
      next = pages_of(t + 2 * NW);
      __builtin_amdgcn_sched_barrier(0);
      ask(kr, kb, ks, kl);
      __builtin_amdgcn_sched_barrier(0);
      // weights: key d = t KT + 16 u + 4 g + e of query r16
      bool whole = t * KT >= all_lo && t * KT + KT - 1 <= all_hi;  // all rows see all keys (wave-uniform)
#pragma unroll
      for (int u = 0; u < SUB; ++u) whole = whole && __ballot(now[u]) == ~0ull;
      u32x4 w[RT], wl[RT];
#pragma unroll
      for (int a = 0; a < RT; ++a) {
        if (!whole) {
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            const uint64_t there = __ballot(now[u]);  // bit r16: key 16 u + r16
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int in = 4 * g + k, d = t * KT + 16 * u + in;
              if (!(d >= lo[a] && d <= hi[a] && (there >> in & 1))) x[a][u][k] = kNone;
            }
          }
        }
        float e[SUB][4], top = kNone;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) top = fmaxf(top, x[a][u][k]);
        top = fmaxf(m[a], fmaf(max_of_groups(top), p.scale, -kTop<ST>));
        const float base = top == kNone ? 0.f : top, keep = __builtin_amdgcn_exp2f(m[a] - base);
        m[a] = top;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            e[u][k] = __builtin_amdgcn_exp2f(fmaf(x[a][u][k], p.scale, -base));
            sum += e[u][k];
          }
        l[a] = fmaf(l[a], keep, sum);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[a][n] *= keep;
        if constexpr (E == 2) {
          float low[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) low[k] = e[k >> 2][k & 3] - round_to<ST>(e[k >> 2][k & 3]);
          w[a] = Tr<ST>::pack(&e[0][0]);
          wl[a] = Tr<ST>::pack(low);
        } else {
          w[a] = Tr<ST>::pack(&e[0][0]);
        }
      }
      // V: a key that is not there gives zeros, since 0 times what memory holds might not be
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int c = 0; c < NB; ++c) {
          u32x4 v = vr[u][c];
          if (!whole && !now[u]) v = u32x4{0u, 0u, 0u, 0u};
          *reinterpret_cast<u32x4*>(stage + (16 * u + r16) * VROW + c * 64 + g * 16) = v;
        }
      __builtin_amdgcn_sched_barrier(0);
      ask(vr, vb, vs, vl);
      __builtin_amdgcn_sched_barrier(0);
      wave_lds_sync();
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (E == 2) {
          typedef short i16x4 __attribute__((ext_vector_type(4)));
          i16x4 v[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            unsigned char* src = stage + (16 * u + 4 * g + (r16 >> 2)) * VROW + (n * 16 + 4 * (r16 & 3)) * 2;
            v[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)src);
          }
          const u32x2 v0 = __builtin_bit_cast(u32x2, v[0]), v1 = __builtin_bit_cast(u32x2, v[1]);
          const u32x4 vt = u32x4{v0.x, v0.y, v1.x, v1.y};
#pragma unroll
          for (int a = 0; a < RT; ++a) {
            o[a][n] = MmaL<ST>::k32(vt, w[a], o[a][n]);
            o[a][n] = MmaL<ST>::k32(vt, wl[a], o[a][n]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float v = *reinterpret_cast<const float*>(stage + (4 * g + k) * VROW + (n * 16 + r16) * 4);
#pragma unroll
            for (int a = 0; a < RT; ++a) o[a][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, __uint_as_float(w[a][k]), o[a][n], 0, 0, 0);
          }
        }
      }
      wave_lds_sync();  // the next tile overwrites the staged rows
    }
  }

  // the waves' parts meet: scaled to the largest maximum, side by side in LDS
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    l[a] = sum_of_groups(l[a]);
    if (!live[a]) {
      m[a] = kNone;
      l[a] = 0.f;
    }
    if (g == 0) ml[wave * ROWS + 16 * a + r16] = part_of(m[a], l[a]);
  }
  __syncthreads();  // and every wave is done with its staged rows
  float* const sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    float top = kNone;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w * ROWS + 16 * a + r16].x);
    const float f = __builtin_amdgcn_exp2f(m[a] - (top == kNone ? 0.f : top));
#pragma unroll
    for (int n = 0; n < NT; ++n)
      *reinterpret_cast<f32x4_t*>(sums + (wave * ROWS + 16 * a + r16) * STRIDE + 16 * n + 4 * g) = live[a] ? o[a][n] * f : f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  attend_end<ST, HD, PAGED, ROWS, NW, 64 * NW, KT>(p, it, s, keys, sums, ml, qs);
}

// ---- many rows

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

// D[a's row][b's row] += a . b over 16 columns: lane (r = lane & 31, h = lane >> 5) holds columns 8 h .. 8 h + 7
// of row r of each, and gets D of rows 8 j + 4 h + e of a (register 4 j + e) with row r of b.
template <typename ST>
__device__ static inline f32x16_t mma32(const u32x4 a, const u32x4 b, const f32x16_t c) {
  typedef typename MmaL<ST>::H8 H8;
  if constexpr (__is_same(ST, bf16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
}

// Where the 16-byte pieces of a row of a staged tile lie: piece c of row r at c ^ mix(r). A product's
// operand reads one piece of 32 rows, the transposed read of V 64 bytes of 8 rows: either then
// meets all banks alike.
template <int HD>
__device__ static inline int mix(int r) {
  if constexpr (HD == 128) return (r & 3) << 2 | (r >> 2 & 3);
  return (r >> 1 & 1) << 2 | (r >> 2 & 3);
}

constexpr float kSlack = 6.f;
template <typename ST>
constexpr float kLift = kTop<ST> > 0.f ? kTop<ST> - kSlack : 0.f;
constexpr uint32_t kNowhere = 0xc0000000u;  // past any resource, also with an instruction's offset: reads zeros

// A buffer resource as four words: `records` bytes from base.
__device__ static inline u32x4 resource_words(const void* base, uint32_t records) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  return u32x4{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, records, 0x00020000u};  // word 3 as bytes_rsrc's
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0, which nothing else here uses, is written
// N loads of 16 bytes a lane: from byte off[i] + 1024 i to lds + 1024 i + 16 lane (lds wave-uniform; an
// instruction's offset counts on both sides). Written as assembly because the compiler waits for every
// load to LDS that it knows of before any read of LDS, which would end the overlap with the tile that
// is worked on; it names no register as output, and wait_vm counts it. s_nop: the cycles that m0, and
// words that vector code may have made, need.
template <int N>
__device__ static inline void stage_bytes(const u32x4 r, uint32_t lds, const uint32_t (&off)[N]) {
  static_assert(N == 2 || N == 4, "16 rows of 128 or 256 bytes");
  if constexpr (N == 2)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\tbuffer_load_dwordx4 %2, %3, 0 offen offset:1024 lds" ::"s"(lds),
                 "v"(off[0]), "v"(off[1]), "s"(r)
                 : "memory", "m0");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\tbuffer_load_dwordx4 %2, %5, 0 offen offset:1024 lds\n\t"
        "buffer_load_dwordx4 %3, %5, 0 offen offset:2048 lds\n\tbuffer_load_dwordx4 %4, %5, 0 offen offset:%6 lds" ::"s"(lds),
        "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(r), "n"(3 * 1024)
        : "memory", "m0");
}
#pragma clang diagnostic pop

// 128 rows of a key head a workgroup, 32 a wave; KG groups of 4 waves take tiles of 64 keys in turn.
// A group stages its tile of K and V in LDS, a tile ahead, straight from memory. As in
// attend_few_kernel products are transposed, so that a lane has one query; the weights are rounded once to
// the type for the second product (half a step of it relative to each; fp16: those below 2^-23 of the largest to 2^-34
// of it). A low part as attend_few_kernel's takes 85 us here instead of 65, for 1.66e-3 from the definition instead of 2.34e-3,
// 1.65e-3 of which are the output's own rounding to bf16: within the type's half step, and not worth a third of the speed.
// 4 x 512 tokens of 16 heads over 4 of 128 behind 3500 earlier ones, 58.7 GFLOP: 64 us (914 TFLOP/s). Bound by no one thing: of
// 68.4 us (an earlier form of the end) 61.6 are left without the weights (exp2, conversions), 63.1 without the operands' reads
// from LDS, 53.7 without both, where a large product's rate is 41.5; the other group's products hide a part of each. With one tile of
// registers between the products 119, staged straight to LDS 113, two groups in turn 81, a wave's loads from one page 73. One group is enough
// where there are 512 workgroups, two of which are on a CU.
template <typename ST, int HD, bool PAGED, int KG>
__global__ void __launch_bounds__(256 * KG, 2) attend_many_kernel(const AttendK<ST> p) {
  constexpr int ROWS = 128, KT = 64, C = HD / 8, RB = HD * 2, NB = HD / 32, NK = HD / 16, RPI = 64 / C, LOADS = 16 / RPI;
  constexpr int kTile = KT * RB, kBuf = 2 * kTile;  // K and V of a tile
  constexpr int STRIDE = HD + 4, kSums = KG * ROWS * STRIDE * 4;
  constexpr int kStage = KG * 2 * kBuf;
  __shared__ __align__(16) unsigned char smem[kStage > kSums ? kStage : kSums];
  __shared__ float2 ml[KG * ROWS];
  __shared__ float qs[4 * KG * HD];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5, wv = wave & 3, kg = wave >> 2;
  StreamOf s;
  const ItemOf it = item_of<ST, PAGED>(p, ROWS, s);
  if (!it.live) return;
  const KeysOf keys = keys_of<ST, PAGED, KT>(p, s, it.row0, ROWS, it.split);

  const int row = it.row0 + 32 * wv + r32;
  u32x4 q[NK];
  int lo, hi;
  {
    const int rr = min(row, p.R - 1), i = rr / p.G;
    const ST* const from = p.q + it.b * p.q_sb + i * p.q_st + (int64_t)(it.hk * p.G + rr - i * p.G) * HD + h * 8;
#pragma unroll
    for (int c = 0; c < NK; ++c) q[c] = ld16(from + c * 16);
    const bool live = row < p.R && i < s.n;
    const int2 seen = seen_by<ST, PAGED>(p, s, i);
    lo = live ? seen.x - keys.k0 : 0;
    hi = live ? seen.y - keys.k0 : -1;
  }
  // what all rows of the wave see, and what some do
  int all_lo = lo, all_hi = hi, some_lo = hi < 0 ? 0x7fffffff : lo, some_hi = hi;
  for (int d = 1; d < 32; d <<= 1) {
    all_lo = max(all_lo, __shfl_xor(all_lo, d));
    all_hi = min(all_hi, __shfl_xor(all_hi, d));
    some_lo = min(some_lo, __shfl_xor(some_lo, d));
    some_hi = max(some_hi, __shfl_xor(some_hi, d));
  }
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  some_lo = __builtin_amdgcn_readfirstlane(some_lo);
  some_hi = __builtin_amdgcn_readfirstlane(some_hi);
  f32x16_t o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[n][e] = 0.f;
  float m = kNone, l = 0.f;

  if (keys.t0 < keys.t1) {
    // What is read goes by offsets that the hardware checks: kNowhere gives zeros, so that 0 times what memory
    // holds for a key that is not there is 0 (its score is 0, too: `weights` takes it out).
    const int32_t* const ring = PAGED ? p.rows + it.b * p.rows_stride + 1 : nullptr;
    // A wave stages rows 16 wv .. 16 wv + 15 of its group's tiles: of one page, since pages have 16 frames or
    // more here and k0 is a multiple of KT, so that a load needs no arithmetic but its page's address.
    // Page of tile t's rows, for tiles in ascending order (the ring entry goes along, so that there is a division
    // only where it wraps). A scalar load: the counts of vector loads are those of the tiles alone.
    uint32_t at_page = 0, at_entry = 0;
    auto page_of = [&](int t) {
      if constexpr (PAGED) {
        const int d = t * KT + 16 * wv;
        if (t >= keys.t1 || d + 15 < keys.lo || d > keys.hi) return -1;
        const uint32_t page = ((uint32_t)keys.k0 + (uint32_t)d) >> p.page_shift;
        at_entry += page - at_page;
        at_page = page;
        if (at_entry >= (uint32_t)p.max_pages) at_entry %= (uint32_t)p.max_pages;
        return (int)reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(ring))[at_entry];
      } else {
        return 0;
      }
    };
    unsigned char* const group = smem + kg * 2 * kBuf;
    const uint32_t group_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)group) + 16 * wv * RB;
    // a lane's byte in the wave's 16 rows, of each load (sources start kBack early, for the instructions' offsets)
    constexpr uint32_t kBack = 1024 * (LOADS - 1);
    uint32_t koff[LOADS], voff[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * RPI + lane / C, c = (lane & (C - 1)) ^ mix<HD>(x);
      koff[i] = kBack - 1024 * i + (PAGED ? (((uint32_t)(c >> 2) << p.page_shift) + x) * 64 + (c & 3) * 16 : (uint32_t)x * (uint32_t)p.k_st + c * 16);
      voff[i] = PAGED ? koff[i] : kBack - 1024 * i + (uint32_t)x * (uint32_t)p.v_st + c * 16;
    }
    const unsigned char* const kb = p.k - kBack + (PAGED ? (int64_t)it.hk * NB << (p.page_shift + 6) : it.b * p.k_sb + (int64_t)it.hk * RB);
    const unsigned char* const vb = p.v - kBack + (PAGED ? (int64_t)it.hk * NB << (p.page_shift + 6) : it.b * p.v_sb + (int64_t)it.hk * RB);
    // where the wave's rows of tile t are: bytes from the base of pages, or the first of the states; -1: nowhere
    auto place_of = [&](int t, int page) -> int64_t {
      const int d = t * KT + 16 * wv;
      if constexpr (PAGED) {
        if ((uint32_t)page >= (uint32_t)p.num_pages) return -1;
        return page * p.page_bytes + ((((uint32_t)keys.k0 + (uint32_t)d) & ((1u << p.page_shift) - 1u)) << 6);
      } else {
        return t < keys.t1 ? d : -1;
      }
    };
    auto ask = [&](bool v, int t, int64_t place, int buf) {
      const int d = t * KT + 16 * wv;
      const int64_t st = v ? p.v_st : p.k_st;
      const u32x4 from = resource_words((v ? vb : kb) + (PAGED ? max(place, (int64_t)0) : max(place, (int64_t)0) * st), PAGED ? 0x7fffffffu : (uint32_t)(15 * st) + RB + kBack);
      const uint32_t to = group_at + buf * kBuf + (v ? kTile : 0);
      if (place >= 0 && d >= keys.lo && d + 15 <= keys.hi) {  // wave-uniform
        stage_bytes<LOADS>(from, to, v ? voff : koff);
      } else {
        uint32_t off[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int x = d + i * RPI + lane / C;
          off[i] = place >= 0 && x >= keys.lo && x <= keys.hi ? (v ? voff[i] : koff[i]) : kNowhere;
        }
        stage_bytes<LOADS>(from, to, off);
      }
    };
    // Pages of the split's keys that are not there (rare): the hardware's zeros would weigh as scores of 0, so their
    // 16 keys are taken out of each tile, by the ring again. Whether there are any is found while the first tiles are on
    // their way, by entries that are asked for before them, and sends each tile by way of the masks then: without absent pages
    // the prompts above take 0.3 us longer than without all of this (a loop that looks here 0.7, a test of its own in each turn 0.9).
    constexpr int LOOK = PAGED ? 4 : 1;
    int32_t look[LOOK];
    const int page0 = PAGED ? (int)(((uint32_t)keys.k0 + (uint32_t)max(keys.lo, keys.t0 * KT)) >> p.page_shift) : 0;
    const int pages = PAGED ? (int)(((uint32_t)keys.k0 + (uint32_t)min(keys.hi, keys.t1 * KT - 1)) >> p.page_shift) - page0 + 1 : 0;
    auto entry_of = [&](int i) { return (uint32_t)(page0 + min(i, pages - 1)) % (uint32_t)p.max_pages; };
    if constexpr (PAGED) {
#pragma unroll
      for (int u = 0; u < LOOK; ++u) look[u] = ring[entry_of(64 * u + lane)];
    }
    bool holes = false;  // wave-uniform
    auto find_holes = [&]() {
      if constexpr (PAGED) {
        bool away = false;
#pragma unroll
        for (int u = 0; u < LOOK; ++u) away |= (uint32_t)look[u] >= (uint32_t)p.num_pages;
        for (int i = 64 * LOOK + lane; i < pages; i += 64) away |= (uint32_t)ring[entry_of(i)] >= (uint32_t)p.num_pages;
        holes = __any(away);
        if (holes) all_hi = -1;  // each tile goes where keys are taken out
      }
    };
    // whether keys d .. d + 15 (wave-uniform, d a multiple of 16) have a page; those that nobody sees have one
    auto there = [&](int d) {
      if (d + 15 < keys.lo || d > keys.hi) return true;
      const uint32_t entry = (((uint32_t)keys.k0 + (uint32_t)d) >> p.page_shift) % (uint32_t)p.max_pages;
      const int32_t page = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(ring))[__builtin_amdgcn_readfirstlane(entry)];
      return (uint32_t)page < (uint32_t)p.num_pages;
    };
    // operand addresses in a tile
    const int kx = mix<HD>(r32);
    int va[2];
    const int l16 = lane & 15, dg = lane >> 4 & 1;
#pragma unroll
    for (int u = 0; u < 2; ++u) va[u] = 8 * u + 4 * h + (l16 >> 2);
    // Scores of a tile from K in buffer b, and the tile before's weights with V in buffer b: a turn's matrix
    // products.
    u32x4 w[4];
    f32x16_t x[2];
    bool weighed = false;  // w holds the weights of the tile before (wave-uniform)
    auto scores = [&](int b) {
      const unsigned char* const kt = group + b * kBuf + r32 * RB;
      u32x4 k[2][4];  // operands of 4 products, asked for 4 ahead
      auto load = [&](int i) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int c = 2 * i + (y >> 1);
          k[i & 1][y] = *reinterpret_cast<const u32x4*>(kt + 32 * RB * (y & 1) + (((2 * c + h) ^ kx) * 16));
        }
      };
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[u][e] = 0.f;
      load(0);
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) {
        if (i + 1 < NK / 2) load(i + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < 4; ++y) x[y & 1] = mma32<ST>(k[i & 1][y], q[2 * i + (y >> 1)], x[y & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto sums_of = [&](int b) {
      const unsigned char* const vt = group + b * kBuf + kTile;
      u32x4 v[2][NB];
      auto load = [&](int k) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          u32x2 part[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int c = (4 * n + 2 * dg + (l16 >> 1 & 1)) ^ mix<HD>(va[u]);
            const unsigned char* src = vt + (16 * k + va[u]) * RB + c * 16 + (l16 & 1) * 8;
            part[u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)src));
          }
          v[k & 1][n] = u32x4{part[0].x, part[0].y, part[1].x, part[1].y};
        }
      };
      load(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k < 3) load(k + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NB; ++n) o[n] = mma32<ST>(v[k & 1][n], w[k], o[n]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto weights = [&](int d0) {
      if (d0 < all_lo || d0 + KT - 1 > all_hi) {
        const uint32_t from = (uint32_t)(d0 + 4 * h - lo), span = (uint32_t)(hi - lo);  // no keys: hi - lo is -1
        const bool none = hi < lo;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (none || from + (32 * u + 8 * j + e) > span) x[u][4 * j + e] = kNone;
            __builtin_amdgcn_sched_barrier(0);  // few conditions at a time in scalar registers
          }
        if (holes) {  // keys 16 y .. 16 y + 15 of the tile are registers 8 (y & 1) .. 8 (y & 1) + 7 of x[y / 2]
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            if (there(d0 + 16 * y)) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[y >> 1][8 * (y & 1) + e] = kNone;
          }
        }
      }
      float top = kNone;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, x[u][e]);
      {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaf(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])), p.scale, -kLift<ST>);
      }
      // the weights' base follows the maximum less kLift in steps of 2^kSlack or more: sums are rescaled in the
      // first tile and hardly ever again, and weights up to 2^(kLift + kSlack) round as well as those up to 1
      if (__any(top > m + kSlack)) {
        top = fmaxf(top, m);
        const float keep = top == kNone ? 1.f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[n] *= keep;
      }
      const float base = m == kNone ? 0.f : m;
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float e[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          e[k] = __builtin_amdgcn_exp2f(fmaf(x[u][k], p.scale, -base));
          part[k & 3] += e[k];
        }
        w[2 * u] = Tr<ST>::pack(e);
        w[2 * u + 1] = Tr<ST>::pack(e + 8);
      }
      l += (part[0] + part[1]) + (part[2] + part[3]);
    };
    auto meet = [&]() {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    // The two groups take turns at the matrix cores: while one multiplies, the other makes weights. A turn of a
    // group: multiply (tile `turn`'s K, the tile before's V) | ask for the tile after next's K and the next one's V,
    // whose buffers are free now, and weigh. So what a turn multiplies was asked for in the turn before
    // the last, and only those loads are waited for. Behind the last tile zeros are asked for.
    auto tile = [&](int turn) { return keys.t0 + kg + turn * KG; };
    const int turns = (keys.t1 - keys.t0 + KG - 1) / KG;
    int64_t at = place_of(tile(0), page_of(tile(0)));
    ask(false, tile(0), at, 0);
    ask(true, tile(0), at, 0);
    at = place_of(tile(1), page_of(tile(1)));  // of the tile whose V is asked for next
    ask(false, tile(1), at, 1);
    int page = page_of(tile(2));
    if (kg == 1) meet();
    wait_vm<0>();
    find_holes();
    auto turn_of = [&](int turn, auto parity) {
      constexpr int b = decltype(parity)::value;
      wait_vm<2 * LOADS>();
      meet();
      const int t = tile(turn);
      const bool idle = t >= keys.t1 || t * KT > some_hi || t * KT + KT - 1 < some_lo;  // wave-uniform
      __builtin_amdgcn_s_setprio(1);
      if (weighed) sums_of(b ^ 1);
      if (!idle) scores(b);
      __builtin_amdgcn_s_setprio(0);
      meet();
      ask(true, tile(turn + 1), at, b ^ 1);
      at = place_of(tile(turn + 2), page);
      ask(false, tile(turn + 2), at, b);
      page = page_of(tile(turn + 3));
      weighed = !idle;
      if (!idle) weights(t * KT);
    };
    for (int turn = 0; turn <= turns; turn += 2) {
      turn_of(turn, std::integral_constant<int, 0>());
      turn_of(turn + 1, std::integral_constant<int, 1>());  // one past the last may be empty
    }
    if (KG == 2 && kg == 0) meet();
    wait_vm<0>();  // what was asked for behind the last tile
  }

  {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (h == 0) ml[kg * ROWS + 32 * wv + r32] = part_of(m, l);
  __syncthreads();  // and every wave is done with the tiles
  float* const sums = reinterpret_cast<float*>(smem);
  float top = kNone;
#pragma unroll
  for (int k = 0; k < KG; ++k) top = fmaxf(top, ml[k * ROWS + 32 * wv + r32].x);
  const float f = __builtin_amdgcn_exp2f(m - (top == kNone ? 0.f : top));
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t v = f32x4_t{o[n][4 * j], o[n][4 * j + 1], o[n][4 * j + 2], o[n][4 * j + 3]};
      *reinterpret_cast<f32x4_t*>(sums + (kg * ROWS + 32 * wv + r32) * STRIDE + 32 * n + 8 * j + 4 * h) = v * f;
    }
  __syncthreads();
  attend_end<ST, HD, PAGED, ROWS, KG, 256 * KG, KT>(p, it, s, keys, sums, ml, qs);
}

// where a row of a join goes
template <typename ST>
__device__ static inline ST* joined_at(const AttendK<ST>& p, uint32_t x, int head_dim) {
  const uint32_t unit = x / (uint32_t)p.R, row = x - unit * (uint32_t)p.R;
  const uint32_t b = unit / (uint32_t)p.Hkv, hk = unit - b * (uint32_t)p.Hkv, i = row / (uint32_t)p.G, gq = row - i * (uint32_t)p.G;
  return p.out + b * p.o_sb + i * p.o_st + (int64_t)(hk * p.G + gq) * head_dim;
}
template <typename ST>
__device__ static inline void put4(ST* to, f32x4_t v) {
  float f[4] = {v[0], v[1], v[2], v[3]};
  if constexpr (sizeof(ST) == 4)
    st16(to, Tr<ST>::pack(f));
  else
    *reinterpret_cast<u32x2*>(to) = pack4<ST>(f);
}

// The splits of a row meet: weights by their maxima, sums over them; bound by the launch and one round trip. Few
// splits: HD / 4 lanes a row, a lane with the splits' four columns at once (12,608 rows of 2 parts: 16 us less than
// a workgroup a row).
constexpr int kFewSplits = 8;
template <typename ST, int HD>
__global__ void __launch_bounds__(256) attend_join_few_kernel(const AttendK<ST> p, uint32_t rows) {
  constexpr int LANES = HD / 4;
  const uint32_t x = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (x >= rows) return;
  const int c = (threadIdx.x & (LANES - 1)) * 4;
  float2 v[kFewSplits];
  f32x4_t part[kFewSplits];
#pragma unroll
  for (int u = 0; u < kFewSplits; ++u) {
    const int64_t at = (int64_t)x * p.splits + min(u, p.splits - 1);
    v[u] = p.ml[at];
    part[u] = *reinterpret_cast<const f32x4_t*>(p.part + at * HD + c);
  }
  float top = kNone, l = 0.f;
#pragma unroll
  for (int u = 0; u < kFewSplits; ++u) top = fmaxf(top, v[u].x);
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kFewSplits; ++u) {
    if (u >= p.splits || v[u].y == 0.f) continue;
    const float w = __builtin_amdgcn_exp2f(v[u].x - top);
    l = fmaf(v[u].y, w, l);
    acc += part[u] * w;
  }
  put4(joined_at(p, x, HD) + c, acc * quotient(top, l));
}

// More: a workgroup a row (16 rows of 120 parts: 4.0 us).
constexpr int kMaxSplits = 256;
template <typename ST, int HD>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendK<ST> p) {
  constexpr int LANES = HD / 4, SIDE = 256 / LANES, AHEAD = 8;  // lanes a split's row, splits at once, turns on their way
  __shared__ float weight[kMaxSplits];
  __shared__ float red[4], total[4];
  __shared__ f32x4_t sums[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t x = blockIdx.x;
  const float2 v = tid < p.splits ? p.ml[(int64_t)x * p.splits + tid] : float2{kNone, 0.f};
  // the parts are on their way while their weights are made; one without keys for the row holds zeros
  const int c = (tid & (LANES - 1)) * 4;
  const float* const from = p.part + (int64_t)x * p.splits * HD + c;
  f32x4_t ahead[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) ahead[u] = *reinterpret_cast<const f32x4_t*>(from + (int64_t)min(tid / LANES + u * SIDE, p.splits - 1) * HD);
  float top = v.x;
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = __builtin_amdgcn_exp2f(v.x - (top == kNone ? 0.f : top));
  weight[tid] = v.y == 0.f ? 0.f : w;
  const float l = group_sum<64>(v.y == 0.f ? 0.f : v.y * w);
  if (lane == 0) total[wave] = l;
  __syncthreads();
  f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    const float ws = weight[tid / LANES + u * SIDE];  // 0 past the splits
    acc += ws == 0.f ? f32x4_t{0.f, 0.f, 0.f, 0.f} : ahead[u] * ws;
  }
#pragma unroll 4
  for (int sp = tid / LANES + AHEAD * SIDE; sp < p.splits; sp += SIDE) acc += *reinterpret_cast<const f32x4_t*>(from + (int64_t)sp * HD) * weight[sp];
  sums[tid] = acc;
  __syncthreads();
  if (tid >= LANES) return;
#pragma unroll
  for (int k = 1; k < SIDE; ++k) acc += sums[tid + k * LANES];
  const float sum = (total[0] + total[1]) + (total[2] + total[3]), inv = quotient(top, sum);
  put4(joined_at(p, x, HD) + c, acc * inv);
}

namespace {

// Rows of `name`: 16-byte aligned, strides whole 16-byte pieces.
template <typename ST>
int rows_ok(const char* what, const char* name, const void* at, int64_t sb, int64_t st) {
  if (!at) return fail(PK_ERR_INVALID, "%s: %s is NULL", what, name);
  if (!aligned16(at) || sb < 0 || st < 0 || sb % Tr<ST>::VEC != 0 || st % Tr<ST>::VEC != 0)
    return fail(PK_ERR_INVALID, "%s: %s needs 16-byte aligned rows and strides >= 0 of whole 16-byte pieces", what, name);
  return PK_OK;
}

// A layer of a pool whose rows are whole heads.
int pool_ok(const char* what, const pk_paged_layout& L, int layer, int head_dim) {
  if (head_dim != 64 && head_dim != 128) return fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (built: 64, 128)", what, head_dim);
  if (!L.k_pool || !L.v_pool || !aligned16(L.k_pool) || !aligned16(L.v_pool))
    return fail(PK_ERR_INVALID, "%s: pools must be non-NULL and 16-byte aligned", what);
  if (L.num_layers <= 0 || layer < 0 || layer >= L.num_layers) return fail(PK_ERR_INVALID, "%s: layer %d out of range [0, %d)", what, layer, L.num_layers);
  if (log2_of(L.page_size) < 0) return fail(PK_ERR_INVALID, "%s: page_size %d is not a power of two", what, L.page_size);
  if (L.num_pages <= 0 || (int64_t)L.num_pages * L.page_size >= (int64_t{1} << 31))
    return fail(PK_ERR_INVALID, "%s: need 0 < num_pages * page_size < 2^31", what);
  if (L.d_model <= 0 || L.d_model % head_dim != 0)
    return fail(PK_ERR_INVALID, "%s: pages of %d columns are not whole heads of %d", what, L.d_model, head_dim);
  // rows of 64 bytes of a layer have 32-bit numbers
  if ((int64_t)L.num_pages * L.page_size * (L.d_model / 16) >= (int64_t{1} << 32))
    return fail(PK_ERR_INVALID, "%s: %d pages of %d x %d are past a layer's 2^32 column blocks", what, L.num_pages, L.page_size, L.d_model);
  return PK_OK;
}

template <typename ST>
int norm_append(const pk_qk_norm_append_args* a, hipStream_t s) {
  const char* what = "pk_qk_norm_append";
  const pk_paged_layout& L = a->pages;
  int rc = pool_ok(what, L, a->layer, a->head_dim);
  if (rc != PK_OK) return rc;
  if (a->batch < 0 || a->chunk < 0 || (int64_t)a->batch * a->chunk >= (int64_t{1} << 31) || a->num_heads <= 0 || a->num_heads > 65536 || L.d_model > (1 << 22))
    return fail(PK_ERR_INVALID, "%s: need batch and chunk >= 0, fewer than 2^31 tokens and 0 < num_heads <= 65536", what);
  if (a->rotary < 0 || (a->rotary > 0 && (log2_of(a->rotary) < 4 || a->rotary > a->head_dim)))
    return fail(PK_ERR_UNSUPPORTED, "%s: rotary %d (built: 0, powers of two from 16 to head_dim)", what, a->rotary);
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return fail(PK_ERR_INVALID, "%s: eps must be >= 0", what);
  if (a->batch == 0 || a->chunk == 0) return PK_OK;
  if ((rc = rows_ok<ST>(what, "query", a->query, a->query_stride_b, a->query_stride_t)) != PK_OK) return rc;
  if ((rc = rows_ok<ST>(what, "key", a->key, a->key_stride_b, a->key_stride_t)) != PK_OK) return rc;
  if ((rc = rows_ok<ST>(what, "value", a->value, a->value_stride_b, a->value_stride_t)) != PK_OK) return rc;
  if ((rc = rows_ok<ST>(what, "out", a->out, a->out_stride_b, a->out_stride_t)) != PK_OK) return rc;
  if ((a->q_weight && !aligned16(a->q_weight)) || (a->k_weight && !aligned16(a->k_weight)))
    return fail(PK_ERR_INVALID, "%s: weights must be 16-byte aligned", what);
  if (!a->slot_map || (a->rotary > 0 && !a->inv_freq) || (a->rotary > 0 && !a->positions && !L.rows))
    return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (a->slot_map_stride_b < 0 || a->positions_stride_b < 0) return fail(PK_ERR_INVALID, "%s: a stride is negative", what);
  NormK<ST> p{};
  const int64_t slab = (int64_t)a->layer * L.num_pages * L.page_size * L.d_model;
  p.q = static_cast<const ST*>(a->query);
  p.k = static_cast<const ST*>(a->key);
  p.v = static_cast<const ST*>(a->value);
  p.out = static_cast<ST*>(a->out);
  p.kp = static_cast<ST*>(L.k_pool) + slab;
  p.vp = static_cast<ST*>(L.v_pool) + slab;
  p.qw = static_cast<const ST*>(a->q_weight);
  p.kw = static_cast<const ST*>(a->k_weight);
  p.inv = a->inv_freq;
  p.pos = a->positions;
  p.pos_sb = a->positions_stride_b;
  p.rows = L.rows;
  p.rows_stride = L.rows_stride;
  p.map = a->slot_map;
  p.map_sb = a->slot_map_stride_b;
  p.q_sb = a->query_stride_b;
  p.q_st = a->query_stride_t;
  p.k_sb = a->key_stride_b;
  p.k_st = a->key_stride_t;
  p.v_sb = a->value_stride_b;
  p.v_st = a->value_stride_t;
  p.o_sb = a->out_stride_b;
  p.o_st = a->out_stride_t;
  p.B = a->batch;
  p.T = a->chunk;
  p.Hq = a->num_heads;
  p.Hkv = L.d_model / a->head_dim;
  p.rotary = a->rotary;
  p.interleaved = a->interleaved ? 1 : 0;
  p.page_shift = log2_of(L.page_size);
  p.places = (uint32_t)L.num_pages << p.page_shift;
  p.eps = a->eps;
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const int64_t total = (int64_t)p.B * p.T;
  // few tokens: one a workgroup, for the shortest chain; many: 4 or 8, whose loads go together. 20 heads of 128 in bf16, us with
  // 1 / 4 / 8: 1024 tokens 5.8 / 7.1 / 10.0, 1536 7.3 / 8.8 / 10.3, 2048 9.9 / 9.6 / 11.0, 4096 14.4 / 12.6 / 12.9, 8192
  // 22.8 / 20.2 / 17.6, 16384 51.2 / 42.1 / 31.7
  const int tok = total <= 1024 ? 1 : total <= 8192 ? 4 : 8;
  const dim3 grid((unsigned)((total + tok - 1) / tok));
  if ((int64_t)grid.x >= (1 << 24)) return fail(PK_ERR_UNSUPPORTED, "%s: %lld tokens in one call (built: fewer than 2^27)", what, (long long)total);
  auto launch = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    if (tok == 1)
      hipLaunchKernelGGL((qk_norm_append_kernel<ST, HD, 1, 2>), grid, dim3(256), 0, s, p);
    else if (tok == 4)
      hipLaunchKernelGGL((qk_norm_append_kernel<ST, HD, 4, 4>), grid, dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((qk_norm_append_kernel<ST, HD, 8, 5>), grid, dim3(256), 0, s, p);
  };
  if (a->head_dim == 64)
    launch(std::integral_constant<int, 64>());
  else
    launch(std::integral_constant<int, 128>());
  return check_launch(what);
}

constexpr float kLog2E = 1.44269504088896341f;

// What both attentions ask of a call.
int attend_ok(const char* what, int batch, int chunk, int heads, int kv_heads, int head_dim, float scale) {
  if (head_dim != 64 && head_dim != 128) return fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (built: 64, 128)", what, head_dim);
  if (batch < 0 || chunk < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return fail(PK_ERR_INVALID, "%s: need batch and chunk >= 0 and whole groups of query heads (got %d, %d, %d over %d)", what, batch, chunk, heads,
                kv_heads);
  if ((int64_t)batch * chunk * heads >= (int64_t{1} << 31)) return fail(PK_ERR_INVALID, "%s: 2^31 rows or more", what);
  if (!(scale > 0.f) || !std::isfinite(scale * kLog2E)) return fail(PK_ERR_INVALID, "%s: scale must be > 0 and finite, times log2(e) too", what);
  return PK_OK;
}

// How a call is cut: rows of a workgroup, workgroups along the rows and along the keys.
struct AttendCut {
  int rows, key_groups, row_tiles, splits;
  int64_t groups;  // workgroups
};

AttendCut attend_cut(int dtype, int batch, int chunk, int heads, int kv_heads, int keys, bool narrow) {
  AttendCut c;
  const int64_t R = (int64_t)chunk * (heads / kv_heads), units = (int64_t)batch * kv_heads;
  // From 33 rows on 128 a workgroup in 16 bits, for batches: 64 x 33 rows of 8 heads of 128 over 1500 states 82.8 us, 110.7
  // with 32; 64 x 48 of 64 over the same 43.4 and 50.8; 64 x 36 of 4 heads of 128 over 3009 tokens 81.3 and 84.0. Few streams of up to
  // 64 rows pay for it, whose keys it splits less: 4 x 48 rows of 8 heads of 64 over 1048 tokens 21.3 us, 13.8 with 32; 32 x 48
  // 28.6 and 22.6; 8 x 36 of 4 heads of 128 over 3009 26.2 and 24.7; 32 x 96 24.3 and 27.5.
  c.rows = R <= 16 ? 16 : R <= 32 || dtype == PK_DTYPE_F32 || narrow ? 32 : 128;
  c.key_groups = c.rows == 128 && units * ((R + 127) / 128) < 512 ? 2 : 1;
  c.row_tiles = (int)((R + c.rows - 1) / c.rows);
  // keys are split over workgroups where the rows leave CUs without one (256 CUs hold one of attend_many_kernel's
  // workgroups each, and two of attend_few_kernel's); a part has 512 keys at least, since parts are joined in a launch
  // of 4 us. So 384 workgroups or more are left whole (128 streams over up to 4096, 512 of them: 88 us whole,
  // 97 in two parts), fewer are not (36 x 4 rows over up to 1500 states, 288: 41.1 us whole, 36.3 in two; 61 streams over up to
  // 4000, 244: 46.3 in two, 50.9 in three)
  const int64_t whole = units * c.row_tiles, full = c.rows == 128 ? 256 : 512;
  int64_t n = std::min((full * 3 / 4 + whole - 1) / whole, (int64_t)keys / 512);
  n = std::min(std::max(n, (int64_t)1), (int64_t)kMaxSplits);
  c.splits = (int)n;
  c.groups = (units * n + 7) / 8 * 8 * c.row_tiles;
  return c;
}

int64_t attend_space(int64_t rows, int splits, int head_dim) { return splits > 1 ? rows * splits * (4 * head_dim + 8) : 0; }

template <typename ST, int HD, bool PAGED>
int attend_launch(const char* what, const AttendK<ST>& p, const AttendCut& c, hipStream_t s) {
  const dim3 grid((unsigned)c.groups), block(256);
  constexpr Source SRC = PAGED ? kPages : kStates;
  if (PAGED && p.page_shift < 4) {
    if (c.rows == 16)
      hipLaunchKernelGGL((attend_few_kernel<ST, HD, kSmallPages, 1, false>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((attend_few_kernel<ST, HD, kSmallPages, 2, false>), grid, block, 0, s, p);
  } else if (c.rows == 16) {
    hipLaunchKernelGGL((attend_few_kernel<ST, HD, SRC, 1, PAGED>), grid, block, 0, s, p);
  } else if (c.rows == 32) {
    if (PAGED && c.row_tiles == 1)
      hipLaunchKernelGGL((attend_few_kernel<ST, HD, SRC, 2, PAGED>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((attend_few_kernel<ST, HD, SRC, 2, false>), grid, block, 0, s, p);
  } else if constexpr (sizeof(ST) == 2) {
    if (c.key_groups == 1)
      hipLaunchKernelGGL((attend_many_kernel<ST, HD, PAGED, 1>), grid, block, 0, s, p);
    else
      hipLaunchKernelGGL((attend_many_kernel<ST, HD, PAGED, 2>), grid, dim3(512), 0, s, p);
  }
  int rc = check_launch(what);
  if (rc != PK_OK || p.splits == 1) return rc;
  const uint32_t rows = (uint32_t)p.B * p.Hkv * p.R;
  if (p.splits <= kFewSplits)
    hipLaunchKernelGGL((attend_join_few_kernel<ST, HD>), dim3((rows + 1024 / HD - 1) / (1024 / HD)), block, 0, s, p, rows);
  else
    hipLaunchKernelGGL((attend_join_kernel<ST, HD>), dim3(rows), block, 0, s, p);
  return check_launch(what);
}

// Both attentions, from the cut on.
template <typename ST, bool PAGED>
int attend(const char* what, AttendK<ST>& p, int dtype, int head_dim, int keys, void* workspace, int device, hipStream_t s) {
  p.G = p.Hq / p.Hkv;
  p.R = p.T * p.G;
  const AttendCut c = attend_cut(dtype, p.B, p.T, p.Hq, p.Hkv, keys, PAGED && p.page_shift < 4);
  p.row_tiles = c.row_tiles;
  p.splits = c.splits;
  // workgroups that have a CU each need no order; two of those of 256 threads are on a CU at once. Few keys do not
  // differ by what finding it costs (5 tokens of 60 streams over up to 516: 15.8 us as they are, 16.5 in order; one
  // of 60 over up to 2001: 31.2 and 26.3; 240 x 4 rows over up to 375 states: 48.0 and 52.7)
  const bool ragged = p.B > 1 && (PAGED || p.lengths) && keys >= (PAGED ? 1024 : 512);
  p.order = !ragged || c.groups <= 256 ? kAsTheyAre : c.groups <= 512 && c.key_groups == 1 ? kFolded : kLongFirst;
  p.key_bits = 32 - __builtin_clz((unsigned)keys | 1);
  const int64_t rows = (int64_t)p.B * p.T * p.Hq;
  // a grid has fewer than 2^32 threads
  if (c.groups >= (1 << 24) || (c.splits > 1 && rows >= (1 << 24))) return fail(PK_ERR_UNSUPPORTED, "%s: %lld rows in one call", what, (long long)rows);
  if (c.splits > 1) {
    if (!workspace || !aligned16(workspace)) return fail(PK_ERR_INVALID, "%s: workspace must be non-NULL and 16-byte aligned", what);
    p.part = static_cast<float*>(workspace);
    p.ml = reinterpret_cast<float2*>(p.part + rows * c.splits * head_dim);
  }
  DeviceGuard dg(device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, device);
  return head_dim == 64 ? attend_launch<ST, 64, PAGED>(what, p, c, s) : attend_launch<ST, 128, PAGED>(what, p, c, s);
}

template <typename ST>
int chunk_attn(const pk_chunk_attn_args* a, hipStream_t s) {
  const char* what = "pk_chunk_attn";
  const pk_paged_layout& L = a->pages;
  int rc = pool_ok(what, L, a->layer, a->head_dim);
  if (rc != PK_OK) return rc;
  if ((rc = attend_ok(what, a->batch, a->chunk, a->num_heads, L.d_model / a->head_dim, a->head_dim, a->scale)) != PK_OK) return rc;
  if (a->left < 0 || L.max_pages <= 0 || L.rows_stride < 1 + L.max_pages || ((int64_t)a->left + a->chunk + L.page_size - 2) / L.page_size + 1 > L.max_pages)
    return fail(PK_ERR_INVALID, "%s: %d ring entries of %d frames do not hold any window of %d + %d (rows_stride %d)", what, L.max_pages, L.page_size,
                a->left, a->chunk, L.rows_stride);
  if (L.page_size > (1 << 20)) return fail(PK_ERR_UNSUPPORTED, "%s: pages of %d frames (built: up to 2^20)", what, L.page_size);
  if ((int64_t)a->left + a->chunk > (1 << 30)) return fail(PK_ERR_INVALID, "%s: a window of more than 2^30 positions", what);
  if (a->batch == 0 || a->chunk == 0) return PK_OK;
  if (!L.rows) return fail(PK_ERR_INVALID, "%s: rows is NULL", what);
  if ((rc = rows_ok<ST>(what, "query", a->query, a->query_stride_b, a->query_stride_t)) != PK_OK) return rc;
  if ((rc = rows_ok<ST>(what, "out", a->out, a->out_stride_b, a->out_stride_t)) != PK_OK) return rc;
  AttendK<ST> p{};
  const int64_t slab = (int64_t)a->layer * L.num_pages * L.page_size * L.d_model;
  p.q = static_cast<const ST*>(a->query);
  p.out = static_cast<ST*>(a->out);
  p.k = reinterpret_cast<const unsigned char*>(static_cast<const ST*>(L.k_pool) + slab);
  p.v = reinterpret_cast<const unsigned char*>(static_cast<const ST*>(L.v_pool) + slab);
  p.q_sb = a->query_stride_b;
  p.q_st = a->query_stride_t;
  p.o_sb = a->out_stride_b;
  p.o_st = a->out_stride_t;
  p.rows = L.rows;
  p.rows_stride = L.rows_stride;
  p.page_bytes = (int64_t)L.page_size * L.d_model * (int64_t)sizeof(ST);
  p.max_pages = L.max_pages;
  p.page_shift = log2_of(L.page_size);
  p.num_pages = L.num_pages;
  p.lengths = a->lengths;
  p.B = a->batch;
  p.T = a->chunk;
  p.Hq = a->num_heads;
  p.Hkv = L.d_model / a->head_dim;
  p.left = a->left;
  p.scale = a->scale * kLog2E;
  return attend<ST, true>(what, p, a->dtype, a->head_dim, a->left + a->chunk, a->workspace, a->device, s);
}

template <typename ST>
int cross_attn(const pk_cross_attn_args* a, hipStream_t s) {
  const char* what = "pk_cross_attn";
  int rc = attend_ok(what, a->batch, a->chunk, a->num_heads, a->kv_heads, a->head_dim, a->scale);
  if (rc != PK_OK) return rc;
  if (a->states < 0 || a->states > (1 << 30)) return fail(PK_ERR_INVALID, "%s: need 0 <= states <= 2^30", what);
  if (a->batch == 0 || a->chunk == 0) return PK_OK;
  if ((rc = rows_ok<ST>(what, "query", a->query, a->query_stride_b, a->query_stride_t)) != PK_OK) return rc;
  if ((rc = rows_ok<ST>(what, "out", a->out, a->out_stride_b, a->out_stride_t)) != PK_OK) return rc;
  if (a->states > 0) {
    if ((rc = rows_ok<ST>(what, "key", a->key, a->key_stride_b, a->key_stride_t)) != PK_OK) return rc;
    if ((rc = rows_ok<ST>(what, "value", a->value, a->value_stride_b, a->value_stride_t)) != PK_OK) return rc;
    // a tile of 64 states is addressed with 32 bits
    if (a->key_stride_t >= (1 << 23) || a->value_stride_t >= (1 << 23)) return fail(PK_ERR_UNSUPPORTED, "%s: rows of 2^23 elements or more", what);
  }
  AttendK<ST> p{};
  constexpr int64_t E = sizeof(ST);
  p.q = static_cast<const ST*>(a->query);
  p.out = static_cast<ST*>(a->out);
  p.k = static_cast<const unsigned char*>(a->key);
  p.v = static_cast<const unsigned char*>(a->value);
  p.q_sb = a->query_stride_b;
  p.q_st = a->query_stride_t;
  p.o_sb = a->out_stride_b;
  p.o_st = a->out_stride_t;
  p.k_sb = a->key_stride_b * E;
  p.k_st = a->key_stride_t * E;
  p.v_sb = a->value_stride_b * E;
  p.v_st = a->value_stride_t * E;
  p.lengths = a->lengths;
  p.B = a->batch;
  p.T = a->chunk;
  p.Hq = a->num_heads;
  p.Hkv = a->kv_heads;
  p.states = a->states;
  p.scale = a->scale * kLog2E;
  return attend<ST, false>(what, p, a->dtype, a->head_dim, a->states, a->workspace, a->device, s);
}

}  // namespace
}  // namespace pk

// the typed call of an entry point
#define PK_BY_DTYPE(name, call)                                                        \
  pk::clear_error();                                                                   \
  if (!args) return pk::fail(PK_ERR_INVALID, name ": args is NULL");                   \
  hipStream_t s = static_cast<hipStream_t>(stream);                                    \
  switch (args->dtype) {                                                               \
    case PK_DTYPE_F32: return pk::call<float>(args, s);                                \
    case PK_DTYPE_F16: return pk::call<_Float16>(args, s);                             \
    case PK_DTYPE_BF16: return pk::call<pk::bf16_t>(args, s);                          \
    default: return pk::fail(PK_ERR_INVALID, name ": unknown dtype %d", args->dtype);  \
  }

extern "C" {

int pk_qk_norm_append(const pk_qk_norm_append_args* args, void* stream) { PK_BY_DTYPE("pk_qk_norm_append", norm_append) }

int64_t pk_attn_workspace_bytes(int32_t dtype, int32_t batch, int32_t chunk, int32_t num_heads, int32_t kv_heads, int32_t head_dim, int32_t keys) {
  if (batch <= 0 || chunk <= 0 || num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads != 0 || head_dim <= 0 || keys < 0) return 0;
  // for pages of any size
  const int a = pk::attend_cut(dtype, batch, chunk, num_heads, kv_heads, keys, false).splits, b = pk::attend_cut(dtype, batch, chunk, num_heads, kv_heads, keys, true).splits;
  return pk::attend_space((int64_t)batch * chunk * num_heads, a > b ? a : b, head_dim);
}

int pk_chunk_attn(const pk_chunk_attn_args* args, void* stream) { PK_BY_DTYPE("pk_chunk_attn", chunk_attn) }

int pk_cross_attn(const pk_cross_attn_args* args, void* stream) { PK_BY_DTYPE("pk_cross_attn", cross_attn) }

}  // extern "C"
