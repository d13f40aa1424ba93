// gfx950 attention of a text decoder: new tokens over a paged cache, and over the encoder's
// states; the norms and rotation of new queries and keys with their way into the pages.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "pk_common.h"
#include "pk_device.h"
#include "pk_scan.h"

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

template <typename ST, int HD, int TOK>
__global__ void __launch_bounds__(256) qk_norm_append_kernel(const NormK<ST> p) {
  constexpr int VEC = Tr<ST>::VEC, LPH = HD / VEC, CB = 64 / (int)sizeof(ST);
  __shared__ float2 cs[TOK][HD / 2];
  const int heads = p.Hq + 2 * p.Hkv, per = heads * LPH, half = p.rotary >> 1;
  const int64_t total = (int64_t)p.B * p.T, first = (int64_t)blockIdx.x * TOK;
  for (int i = threadIdx.x; i < TOK * half; i += 256) {
    const int t = i / half, f = i - t * half;
    const int64_t row = first + t;
    if (row < total) {
      const int b = (int)(row / p.T), at = (int)(row - (int64_t)b * p.T);
      const int32_t pos = p.pos ? p.pos[b * p.pos_sb + at] : p.rows[b * p.rows_stride] + at;
      cs[t][f] = turn_of(pos, p.inv[f]);
    }
  }
  __syncthreads();
  // columns of a token in order: the heads of q, k and v
  const int all = TOK * per;
  for (int i0 = 0; i0 < all; i0 += 256) {
    const int i = min(i0 + (int)threadIdx.x, all - 1);  // every lane takes part in the sums
    const int t = i / per, j = i - t * per, head = j / LPH, c = (j - head * LPH) * VEC;
    const int64_t row = first + t;
    bool live = i0 + (int)threadIdx.x < all && row < total;
    const int b = live ? (int)(row / p.T) : 0, at = live ? (int)(row - (int64_t)b * p.T) : 0;
    const int which = head < p.Hq ? 0 : head < p.Hq + p.Hkv ? 1 : 2;
    const int h = which == 0 ? head : which == 1 ? head - p.Hq : head - p.Hq - p.Hkv;
    ST* to = nullptr;
    if (which == 0) {
      to = p.out + b * p.o_sb + at * p.o_st + (int64_t)h * HD + c;
    } else if (live) {
      const uint32_t place = (uint32_t)p.map[b * p.map_sb + at];
      live = place < p.places;
      const int col = h * HD + c, mask = (1 << p.page_shift) - 1;
      const int64_t e = (int64_t)(place >> p.page_shift) * (((int64_t)p.Hkv * HD) << p.page_shift) +
                        (int64_t)(col / CB) * (CB << p.page_shift) + (int64_t)(place & mask) * CB + col % CB;
      to = (which == 1 ? p.kp : p.vp) + e;
    }
    const ST* const from = which == 0   ? p.q + b * p.q_sb + at * p.q_st + (int64_t)h * HD + c
                           : which == 1 ? p.k + b * p.k_sb + at * p.k_st + (int64_t)h * HD + c
                                        : p.v + b * p.v_sb + at * p.v_st + (int64_t)h * HD + c;
    u32x4 raw = u32x4{0u, 0u, 0u, 0u};
    if (live) raw = ld16(from);
    float x[VEC];
    Tr<ST>::unpack(raw, x);
    const ST* const w = which == 0 ? p.qw : p.kw;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) ss = fmaf(x[e], x[e], ss);
    ss = group_sum<LPH>(ss);
    if (w && which < 2) {
      const float r = 1.f / sqrtf(ss * (1.f / HD) + p.eps);
      float g[VEC];
      Tr<ST>::unpack(ld16(w + c), g);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = x[e] * r * g[e];
    }
    if (p.interleaved) {
      if (which < 2 && c < p.rotary) {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          const float2 f = cs[t][(c + e) >> 1];
          const float a = x[e], z = x[e + 1];
          x[e] = a * f.x - z * f.y;
          x[e + 1] = z * f.x + a * f.y;
        }
      }
    } else if (half > 0) {
      const int span = half / VEC;  // lanes, a power of two
      const bool turned = which < 2 && c < p.rotary, upper = c >= half;
      const int f0 = upper ? c - half : c;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float other = __shfl_xor(x[e], span);
        if (turned) {
          const float2 f = cs[t][f0 + e];
          x[e] = upper ? x[e] * f.x + other * f.y : x[e] * f.x - other * f.y;
        }
      }
    }
    if (live) st16(to, which == 2 ? raw : Tr<ST>::pack(x));
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
};

constexpr float kNone = -__builtin_inff();

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
// scores, columns over the lanes for the sums. q: the row, in fp32, in LDS. Gives the
// maximum (log2 units), the sum, and the sums of columns lane + 64 c.
template <typename ST, int HD, bool PAGED>
__device__ static inline void attend_row(const AttendK<ST>& p, int b, int h, const float* q, int first, int last, float& m, float& l,
                                         float (&acc)[HD / 64]) {
  constexpr int VEC = Tr<ST>::VEC, CB = 64 / (int)sizeof(ST), E = (int)sizeof(ST);
  const int lane = threadIdx.x & 63;
  const int64_t step = PAGED ? (int64_t)64 << p.page_shift : 64;
  m = kNone;
  l = 0.f;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) acc[c] = 0.f;
  const int n = last - first + 1;  // at most 2^30: positions run up to 2^31 - 1, so numbers from `first` on are counted
  for (int d0 = 0; d0 < n; d0 += 64) {
    const int64_t at = d0 + lane < n ? key_at<ST, PAGED>(p, b, HD * E, h, first + d0 + lane, false) : -1;
    float s = kNone;
    if (at >= 0) {
      float d = 0.f;
      for (int c = 0; c < HD; c += VEC) {
        float x[VEC];
        Tr<ST>::unpack(*reinterpret_cast<const u32x4*>(p.k + at + c / CB * step + c % CB * E), x);
#pragma unroll
        for (int e = 0; e < VEC; ++e) d = fmaf(x[e], q[c + e], d);
      }
      s = d * p.scale;
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
    for (int u = 0; u < 64 && d0 + u < n; ++u) {
      const float w = __shfl(e, u);
      const int64_t va = key_at<ST, PAGED>(p, b, HD * E, h, first + d0 + u, true);
      if (va < 0) continue;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const int col = lane + 64 * c;
        acc[c] = fmaf(w, from_st(*reinterpret_cast<const ST*>(p.v + va + col / CB * step + col % CB * E)), acc[c]);
      }
    }
  }
}

template <typename ST, int HD, bool PAGED>
__global__ void __launch_bounds__(256) attend_rows_kernel(const AttendK<ST> p) {
  __shared__ float qs[4][HD];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= (int64_t)p.B * p.T * p.Hq) return;
  const int h = (int)(row % p.Hq), i = (int)(row / p.Hq % p.T), b = (int)(row / p.Hq / p.T);
  const ST* const q = p.q + b * p.q_sb + i * p.q_st + (int64_t)h * HD;
  for (int c = lane; c < HD; c += 64) qs[wave][c] = from_st(q[c]);
  wave_lds_sync();
  const StreamOf s = stream_of<ST, PAGED>(p, b);
  float m = kNone, l = 0.f, acc[HD / 64];
  const int2 seen = seen_by<ST, PAGED>(p, s, i);
  attend_row<ST, HD, PAGED>(p, b, h / p.G, qs[wave], i < s.n ? seen.x : 0, i < s.n ? seen.y : -1, m, l, acc);
  ST* const o = p.out + b * p.o_sb + i * p.o_st + (int64_t)h * HD;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) o[lane + 64 * c] = to_st<ST>(l == 0.f ? 0.f : acc[c] / l);
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
  const dim3 grid((unsigned)total);
  if (a->head_dim == 64)
    hipLaunchKernelGGL((qk_norm_append_kernel<ST, 64, 1>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((qk_norm_append_kernel<ST, 128, 1>), grid, dim3(256), 0, s, p);
  return check_launch(what);
}

// What both attentions ask of a call.
int attend_ok(const char* what, int batch, int chunk, int heads, int kv_heads, int head_dim, float scale) {
  if (head_dim != 64 && head_dim != 128) return fail(PK_ERR_UNSUPPORTED, "%s: head_dim %d (built: 64, 128)", what, head_dim);
  if (batch < 0 || chunk < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return fail(PK_ERR_INVALID, "%s: need batch and chunk >= 0 and whole groups of query heads (got %d, %d, %d over %d)", what, batch, chunk, heads,
                kv_heads);
  if ((int64_t)batch * chunk * heads >= (int64_t{1} << 31)) return fail(PK_ERR_INVALID, "%s: 2^31 rows or more", what);
  if (!(scale > 0.f) || !std::isfinite(scale)) return fail(PK_ERR_INVALID, "%s: scale must be > 0 and finite", what);
  return PK_OK;
}

template <typename ST, bool PAGED>
int attend_launch(const char* what, const AttendK<ST>& p, int head_dim, hipStream_t s) {
  const int64_t rows = (int64_t)p.B * p.T * p.Hq;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (head_dim == 64)
    hipLaunchKernelGGL((attend_rows_kernel<ST, 64, PAGED>), grid, dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((attend_rows_kernel<ST, 128, PAGED>), grid, dim3(256), 0, s, p);
  return check_launch(what);
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
  p.G = p.Hq / p.Hkv;
  p.left = a->left;
  p.scale = a->scale * 1.44269504088896341f;
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  return attend_launch<ST, true>(what, p, a->head_dim, s);
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
  p.G = p.Hq / p.Hkv;
  p.states = a->states;
  p.scale = a->scale * 1.44269504088896341f;
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  return attend_launch<ST, false>(what, p, a->head_dim, s);
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

int64_t pk_attn_workspace_bytes(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

int pk_chunk_attn(const pk_chunk_attn_args* args, void* stream) { PK_BY_DTYPE("pk_chunk_attn", chunk_attn) }

int pk_cross_attn(const pk_cross_attn_args* args, void* stream) { PK_BY_DTYPE("pk_cross_attn", cross_attn) }

}  // extern "C"
