// gfx950 tables of a batch, built on the GPU from what each stream asks for:
//
//   page_step_kernel     block-table rows and slot map of a step from the streams'
//                        slots and frame counts, on a page pool kept in device
//                        memory (the discipline of page_pool.cpp)
//   adapter_plan_kernel  the batch's rows grouped by low-rank adapter

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pk_common.h"
#include "pk_device.h"

namespace pk {

// ---------------------------------------------------------------------------
// page step
//
// With window = left + chunk a slot that has A frames holds the logical pages
//   lo(A) = max(0, A - window) / P  ..  hi(A) = ceil(A / P)   (hi exclusive),
// ring entry k % M, M entries.  Appending n <= chunk frames gives the pages
// lo(A) .. lo(A + n) back and takes hi(A) .. hi(A + n); lo(A + n) <= hi(A), since
// A + n - window <= A.  A pool of at least num_slots * M pages never runs dry, so a
// page given back in a call stands behind every page that the call takes from the
// queue's front or is itself reached in order: all pushes, then all pops at the
// prefix sums over the streams, give the queue that the streams one by one give.

struct PageK {
  int32_t* queue;
  int32_t* head;  // {first entry, entries}
  int64_t* appended;
  int32_t* ring;
  const int32_t* slots;
  const int32_t* lengths;  // or nullptr: chunk each
  int32_t* rows;
  int32_t* slot_map;
  int64_t map_stride;
  int32_t n, S, total, M, page_shift, chunk, rows_stride;
  int32_t window;
  int32_t reset;  // give every page of the slots back instead
};

// inclusive sum over the 64 lanes of a wave
__device__ static inline uint32_t wave_scan(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)v, d);
    if (lane >= d) v += u;
  }
  return v;
}

// exclusive sum over a workgroup of NW waves; `sum`: of all
template <int NW>
__device__ static inline uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t& sum) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t inc = wave_scan(v);
  if (lane == 63) lds[wave] = inc;
  __syncthreads();
  uint32_t before = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const uint32_t x = lds[w];
    if (w < wave) before += x;
    sum += x;
  }
  __syncthreads();
  return before + inc - v;
}

constexpr int kStepThreads = 1024;

struct StreamPages {
  int64_t A;
  int32_t slot;  // -1: absent (out of range, or named before in the call)
  int32_t len, freed, taken, lm, hm;  // ring entries of pages lo and hi
};

__device__ static inline StreamPages stream_pages(const PageK& p, int b, const uint32_t* dup) {
  StreamPages r{};
  const int32_t slot = p.slots[b];
  r.slot = -1;
  if ((uint32_t)slot >= (uint32_t)p.S) return r;
  if (dup[slot >> 5] >> (slot & 31) & 1) {  // rare: the first of equal slots has the step
    for (int j = 0; j < b; ++j)
      if (p.slots[j] == slot) return r;
  }
  const int64_t a = p.appended[slot];
  r.slot = slot;
  r.A = a > 0 ? a : 0;
  const int32_t want = p.lengths ? p.lengths[b] : p.chunk;
  r.len = p.reset ? 0 : min(max(want, 0), p.chunk);
  const int64_t P = (int64_t)1 << p.page_shift, end = r.A + r.len;
  const int64_t w0 = r.A - p.window, w1 = end - p.window;
  const int64_t lo = w0 > 0 ? w0 >> p.page_shift : 0, lo2 = w1 > 0 ? w1 >> p.page_shift : 0;
  const int64_t hi = (r.A + P - 1) >> p.page_shift, hi2 = (end + P - 1) >> p.page_shift;
  r.freed = (int32_t)((p.reset ? hi : lo2) - lo);
  r.taken = (int32_t)(hi2 - hi);
  r.hm = (int32_t)((uint64_t)hi % (uint32_t)p.M);
  r.lm = r.hm - (int32_t)(hi - lo);
  if (r.lm < 0) r.lm += p.M;
  return r;
}

__global__ void __launch_bounds__(kStepThreads) page_step_kernel(const PageK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint32_t sums[kStepThreads / 64];
  const int words = (p.S + 31) >> 5;
  uint32_t* const seen = lds;
  uint32_t* const dup = lds + words;
  const int tid = threadIdx.x;
  for (int i = tid; i < 2 * words; i += kStepThreads) lds[i] = 0;
  const int per = (p.n + kStepThreads - 1) / kStepThreads;
  const int b0 = min(tid * per, p.n), b1 = min(b0 + per, p.n);
  __syncthreads();
  for (int b = b0; b < b1; ++b) {
    const int32_t s = p.slots[b];
    if ((uint32_t)s >= (uint32_t)p.S) continue;
    const uint32_t bit = 1u << (s & 31);
    if (atomicOr(&seen[s >> 5], bit) & bit) atomicOr(&dup[s >> 5], bit);
  }
  __syncthreads();
  uint32_t f = 0, t = 0;
  for (int b = b0; b < b1; ++b) {
    const StreamPages s = stream_pages(p, b, dup);
    f += s.freed;
    t += s.taken;
  }
  uint32_t fsum, tsum;
  f = block_scan<kStepThreads / 64>(f, sums, fsum);
  t = block_scan<kStepThreads / 64>(t, sums, tsum);
  const uint32_t total = (uint32_t)p.total, first = (uint32_t)p.head[0] % total, count = (uint32_t)p.head[1];
  uint32_t at = first + count % total + f;
  for (int b = b0; b < b1; ++b) {
    const StreamPages s = stream_pages(p, b, dup);
    int32_t* const ring = p.ring + (int64_t)s.slot * p.M;
    for (int i = 0; i < s.freed; ++i) {
      int r = s.lm + i;
      if (r >= p.M) r -= p.M;
      p.queue[at++ % total] = ring[r];
      ring[r] = -1;
    }
  }
  __syncthreads();  // every page given back is in the queue
  at = first + t;
  const int P1 = (1 << p.page_shift) - 1;
  for (int b = b0; b < b1; ++b) {
    const StreamPages s = stream_pages(p, b, dup);
    int32_t* const ring = p.ring + (int64_t)s.slot * p.M;
    for (int i = 0; i < s.taken; ++i) {
      int r = s.hm + i;
      if (r >= p.M) r -= p.M;
      ring[r] = p.queue[at++ % total];
    }
    if (!p.reset) {
      int32_t* const row = p.rows + (int64_t)b * p.rows_stride;
      int32_t* const map = p.slot_map + b * p.map_stride;
      row[0] = (int32_t)s.A;
      for (int r = 0; r < p.M; ++r) row[1 + r] = s.slot < 0 ? -1 : ring[r];
      const int64_t hi = (s.A + P1) >> p.page_shift;
      for (int i = 0; i < p.chunk; ++i) {
        const int64_t pos = s.A + i;
        int r = s.hm + (int)((pos >> p.page_shift) - hi);  // -1: the page that A ends in
        r = r < 0 ? r + p.M : r >= p.M ? r - p.M : r;
        map[i] = i < s.len ? (ring[r] << p.page_shift) + (int)(pos & P1) : -1;
      }
    }
  }
  __syncthreads();  // every stream's frame count was read
  for (int b = b0; b < b1; ++b) {
    const StreamPages s = stream_pages(p, b, dup);
    if (s.slot >= 0) p.appended[s.slot] = p.reset ? 0 : s.A + s.len;
  }
  if (tid == 0) {
    p.head[0] = (int32_t)((first + tsum) % total);
    p.head[1] = (int32_t)(count + fsum - tsum);
  }
}

// ---------------------------------------------------------------------------
// adapter plan
//
// A stable counting sort of the streams by adapter in one workgroup: each wave
// counts a run of the streams (LDS), the counts are summed over waves and adapters,
// and each wave places its run in order, 64 streams at a time, a stream's rank among
// the equal ones of its 64 found with one ballot a bit of the number.  Streams
// without an adapter are bucket G.

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kPlanTile = 32;  // rows of a tile

struct PlanK {
  const int32_t* ids;
  int32_t* order;
  int32_t* sorted;
  int4* tiles;
  int32_t B, T, G, max_tiles, bits;
};

__global__ void __launch_bounds__(kPlanThreads) adapter_plan_kernel(const PlanK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint32_t sums[kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int G1 = p.G + 1;
  uint32_t* const hist = lds;                       // [waves][G + 1]
  uint32_t* const start = hist + kPlanWaves * G1;   // [G + 2] first stream of a bucket
  uint32_t* const tile0 = start + G1 + 1;           // [G + 1] first tile of an adapter
  for (int i = tid; i < kPlanWaves * G1; i += kPlanThreads) hist[i] = 0;
  const int run = ((p.B + kPlanWaves - 1) / kPlanWaves + 63) & ~63;
  const int b0 = min(wave * run, p.B), b1 = min(b0 + run, p.B);
  __syncthreads();
  for (int b = b0 + lane; b < b1; b += 64) {
    const int32_t id = p.ids[b];
    atomicAdd(&hist[wave * G1 + ((uint32_t)id < (uint32_t)p.G ? id : p.G)], 1u);
  }
  __syncthreads();
  // bucket g's streams before each wave's, and before bucket g
  uint32_t carry = 0, tcarry = 0;
  for (int g0 = 0; g0 < G1; g0 += kPlanThreads) {
    const int g = g0 + tid;
    uint32_t c = 0;
    if (g < G1)
      for (int w = 0; w < kPlanWaves; ++w) {
        const uint32_t h = hist[w * G1 + g];
        hist[w * G1 + g] = c;
        c += h;
      }
    const uint32_t tiles = g < p.G ? (c * p.T + kPlanTile - 1) / kPlanTile : 0;
    uint32_t all, tall;
    const uint32_t s = block_scan<kPlanWaves>(c, sums, all) + carry;
    const uint32_t t = block_scan<kPlanWaves>(tiles, sums, tall) + tcarry;
    if (g < G1) {
      start[g] = s;
      tile0[g] = t;
      for (int w = 0; w < kPlanWaves; ++w) hist[w * G1 + g] += s;
    }
    carry += all;
    tcarry += tall;
  }
  __syncthreads();
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int b = b0; b < b1; b += 64) {
    const bool in = b + lane < b1;
    const int32_t id = in ? p.ids[b + lane] : -1;
    const bool has = (uint32_t)id < (uint32_t)p.G;
    const int g = has ? id : p.G;
    uint64_t same = __ballot(in);
    for (int i = 0; i < p.bits; ++i) {
      const uint64_t m = __ballot((g >> i) & 1);
      same &= (g >> i) & 1 ? m : ~m;
    }
    uint32_t* const h = &hist[wave * G1 + g];
    uint32_t base = 0;
    if (in) base = *h;
    wave_lds_sync();
    if (in && (same >> lane) == 1) *h = base + __popcll(same);  // the last of the equal ones
    wave_lds_sync();
    if (in) {
      const int64_t at = (int64_t)(base + __popcll(same & below)) * p.T;
      for (int t = 0; t < p.T; ++t) {
        p.order[at + t] = (b + lane) * p.T + t;
        p.sorted[at + t] = has ? id : -1;
      }
    }
  }
  // tile t: the adapter whose tiles it is among (bisection over their first tiles)
  for (int t = tid; t < p.max_tiles; t += kPlanThreads) {
    int4 v = {-1, 0, 0, 0};
    if ((uint32_t)t < tcarry) {
      int lo = 0, hi = p.G;  // tile0[lo] <= t < tile0[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile0[mid] <= (uint32_t)t)
          lo = mid;
        else
          hi = mid;
      }
      const int off = (t - (int)tile0[lo]) * kPlanTile;
      v.x = lo;
      v.y = (int)start[lo] * p.T + off;
      v.z = min(kPlanTile, (int)(start[lo + 1] - start[lo]) * p.T - off);
    }
    p.tiles[t] = v;
  }
}

namespace {

int log2_of(int32_t x) {
  for (int s = 0; s < 31; ++s)
    if ((int32_t{1} << s) == x) return s;
  return -1;
}

int page_step(const pk_page_step_args* a, hipStream_t s) {
  const char* what = "pk_page_step";
  const int ps = log2_of(a->page_size);
  if (ps < 0) return fail(PK_ERR_INVALID, "%s: page_size %d is not a power of two", what, a->page_size);
  if (a->left < 0 || a->chunk <= 0 || a->num_slots <= 0 || a->num_pages <= 0 || a->batch < 0 ||
      (int64_t)a->left + a->chunk + a->page_size >= (int64_t{1} << 31))
    return fail(PK_ERR_INVALID, "%s: need left >= 0, chunk, num_slots and num_pages > 0, batch >= 0 (got %d, %d, %d, %d, %d)", what,
                a->left, a->chunk, a->num_slots, a->num_pages, a->batch);
  const int32_t M = (a->left + a->chunk + a->page_size - 2) / a->page_size + 1;
  if ((int64_t)a->num_pages < (int64_t)a->num_slots * M)
    return fail(PK_ERR_INVALID, "%s: %d pages cannot hold %d slots of %d pages each", what, a->num_pages, a->num_slots, M);
  if (((int64_t)a->num_pages << ps) >= (int64_t{1} << 31) || a->num_pages >= (1 << 30))
    return fail(PK_ERR_INVALID, "%s: %d pages of %d frames are past a slot map's 2^31 frames", what, a->num_pages, a->page_size);
  if (a->num_slots > PK_PAGE_STEP_MAX_SLOTS)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d slots (built: up to %d)", what, a->num_slots, PK_PAGE_STEP_MAX_SLOTS);
  if (a->batch == 0) return PK_OK;
  if (!a->queue || !a->head || !a->appended || !a->ring || !a->slots)
    return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (!a->reset) {
    if (!a->rows || !a->slot_map) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
    if (a->rows_stride < 1 + M || a->slot_map_stride < a->chunk)
      return fail(PK_ERR_INVALID, "%s: need rows_stride >= %d and slot_map_stride >= %d", what, 1 + M, a->chunk);
  }
  PageK k{};
  k.queue = a->queue;
  k.head = a->head;
  k.appended = a->appended;
  k.ring = a->ring;
  k.slots = a->slots;
  k.lengths = a->lengths;
  k.rows = a->rows;
  k.slot_map = a->slot_map;
  k.map_stride = a->slot_map_stride;
  k.n = a->batch;
  k.S = a->num_slots;
  k.total = a->num_pages;
  k.M = M;
  k.page_shift = ps;
  k.chunk = a->chunk;
  k.rows_stride = a->rows_stride;
  k.window = a->left + a->chunk;
  k.reset = a->reset ? 1 : 0;
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const size_t bits = (size_t)((k.S + 31) / 32) * 8;
  hipLaunchKernelGGL(page_step_kernel, dim3(1), dim3(kStepThreads), bits, s, k);
  return check_launch(what);
}

int adapter_plan(const pk_adapter_plan_args* a, hipStream_t s) {
  const char* what = "pk_adapter_plan";
  if (a->batch < 0 || a->frames <= 0 || a->num_adapters <= 0 || (int64_t)a->batch * a->frames >= (int64_t{1} << 31))
    return fail(PK_ERR_INVALID, "%s: need batch >= 0, frames and num_adapters > 0, and fewer than 2^31 rows (got %d, %d, %d)", what,
                a->batch, a->frames, a->num_adapters);
  if (a->num_adapters > PK_ADAPTER_MAX)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d adapters (built: up to %d)", what, a->num_adapters, PK_ADAPTER_MAX);
  const int64_t need = pk_adapter_plan_tiles(a->batch, a->frames, a->num_adapters);
  if (a->max_tiles < need) return fail(PK_ERR_INVALID, "%s: %d tiles, needs %d", what, a->max_tiles, (int)need);
  if (a->batch == 0) return PK_OK;
  if (!a->ids || !a->order || !a->sorted_ids || !a->tiles) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (!aligned16(a->tiles)) return fail(PK_ERR_INVALID, "%s: tiles must be 16-byte aligned", what);
  PlanK k{};
  k.ids = a->ids;
  k.order = a->order;
  k.sorted = a->sorted_ids;
  k.tiles = reinterpret_cast<int4*>(a->tiles);
  k.B = a->batch;
  k.T = a->frames;
  k.G = a->num_adapters;
  k.max_tiles = a->max_tiles;
  while ((1 << k.bits) <= k.G) ++k.bits;
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const size_t lds = sizeof(uint32_t) * ((size_t)kPlanWaves * (k.G + 1) + 2 * (k.G + 2));
  hipLaunchKernelGGL(adapter_plan_kernel, dim3(1), dim3(kPlanThreads), lds, s, k);
  return check_launch(what);
}

}  // namespace
}  // namespace pk

extern "C" int pk_page_step(const pk_page_step_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_page_step: args is NULL");
  return pk::page_step(args, static_cast<hipStream_t>(stream));
}

extern "C" int pk_adapter_plan_tiles(int32_t batch, int32_t frames, int32_t num_adapters) {
  if (batch <= 0 || frames <= 0 || num_adapters <= 0) return 0;
  return (int)((int64_t)batch * frames / pk::kPlanTile + (num_adapters < batch ? num_adapters : batch));
}

extern "C" int pk_adapter_plan(const pk_adapter_plan_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_adapter_plan: args is NULL");
  return pk::adapter_plan(args, static_cast<hipStream_t>(stream));
}
