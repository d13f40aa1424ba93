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

// what rows and slot map need of a stream
struct StepOf {
  int32_t A, slot, len;  // slot -1: absent
  uint32_t at;           // pages taken before the stream's
};

struct PageK {
  int32_t* queue;
  int32_t* head;  // {first entry, entries}
  int64_t* appended;
  int32_t* ring;
  const int32_t* slots;
  const int32_t* lengths;  // or nullptr: chunk each
  int32_t* rows;
  int32_t* slot_map;  // or nullptr
  int64_t map_stride;
  int32_t n, S, total, M, page_shift, chunk, rows_stride;
  int32_t window;
  int32_t reset;  // give every page of the slots back instead
  StepOf* of;  // more than kStepOne streams: [n]
  uint32_t* front;
  uint2* part;  // more than kStepTwo: [n] pages given back and taken
  uint2* sum;   // and of each 256 streams, then of those before them
};

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

constexpr int kStepThreads = 1024;
// Streams of a step in one launch (64 take 8.0 us in a graph so and 8.8 in two, 128 12 and
// 10.1) and in two (2048 take 12.7 us so and 15.3 in four, 4096 16.8 and 15.7, 16384 51 and 18)
constexpr int kStepOne = 64, kStepTwo = 3500;

struct StreamPages {
  uint32_t A;
  int32_t slot;  // -1: absent (out of range, or named before in the call)
  int32_t len, freed, taken;
  uint32_t lo;  // first logical page held
};

// Bits of the slots that the call names twice (LDS, for the workgroup).
template <int V>
__device__ static inline const uint32_t* mark_slots(const PageK& p, uint32_t* lds) {
  const int words = (p.S + 31) >> 5;
  uint32_t* const seen = lds;
  uint32_t* const dup = lds + words;
  for (int i = threadIdx.x; i < 2 * words; i += kStepThreads) lds[i] = 0;
  __syncthreads();
  for (int b0 = 0; b0 < p.n; b0 += kStepThreads * V) {
    int32_t s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int b = b0 + v * kStepThreads + threadIdx.x;
      s[v] = b < p.n ? p.slots[b] : -1;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if ((uint32_t)s[v] >= (uint32_t)p.S) continue;
      const uint32_t bit = 1u << (s[v] & 31);
      if (atomicOr(&seen[s[v] >> 5], bit) & bit) atomicOr(&dup[s[v] >> 5], bit);
    }
  }
  __syncthreads();
  return dup;
}

// the first of equal slots has the step (rare: a search of the streams before, 8 at a time)
__device__ static inline bool named_before(const PageK& p, int b, int32_t slot, const uint32_t* dup) {
  if ((uint32_t)slot >= (uint32_t)p.S || !(dup[slot >> 5] >> (slot & 31) & 1)) return false;
  for (int j = 0; j < b; j += 8) {
    bool hit = false;
#pragma unroll
    for (int u = 0; u < 8; ++u) hit |= p.slots[min(j + u, b - 1)] == slot;
    if (hit) return true;
  }
  return false;
}

// n pages of a slot, ring entry r on, to place `at` of the queue on; e0: the first one's
// number where it is at hand
__device__ static inline void give_back(const PageK& p, int32_t slot, int n, uint32_t r, uint32_t at, const int32_t* e0) {
  int32_t* const ring = p.ring + (int64_t)slot * p.M;
  for (int i = 0; i < n; ++i) {
    p.queue[at] = i == 0 && e0 ? *e0 : ring[r];
    ring[r] = -1;
    if (++r == (uint32_t)p.M) r = 0;
    if (++at == (uint32_t)p.total) at = 0;
  }
}

// dup: nullptr where equal slots are looked for later
__device__ static inline StreamPages stream_pages(const PageK& p, int b, int32_t slot, int32_t want, int64_t a, const uint32_t* dup) {
  StreamPages r{};
  r.slot = -1;
  if ((uint32_t)slot >= (uint32_t)p.S || (dup && named_before(p, b, slot, dup))) return r;
  r.slot = slot;
  r.A = (uint32_t)min(max(a, (int64_t)0), (int64_t)0x7fffffff);
  r.len = p.reset ? 0 : min(max(want, 0), p.chunk);
  const uint32_t P1 = (1u << p.page_shift) - 1u, end = r.A + r.len;  // below 2^32
  const uint32_t lo2 = end > (uint32_t)p.window ? (end - p.window) >> p.page_shift : 0;
  const uint32_t hi = (r.A >> p.page_shift) + ((r.A & P1) != 0), hi2 = (end >> p.page_shift) + ((end & P1) != 0);
  r.lo = r.A > (uint32_t)p.window ? (r.A - p.window) >> p.page_shift : 0;
  r.freed = (int32_t)((p.reset ? hi : lo2) - r.lo);
  r.taken = (int32_t)(hi2 - hi);
  return r;
}

// The streams' part of a step that has to be in order, by one workgroup: who is absent,
// the sums over the streams, the pages given back, the frame counts.  1024 V streams a
// turn, V neighbours a lane: a turn is one chain of round trips (slots, frame counts, the
// sum over the workgroup, rings).
template <int V>
__device__ static inline void step_scan(const PageK& p, uint32_t* lds, uint64_t* sums, StepOf* of, uint32_t& front) {
  const int tid = threadIdx.x;
  const uint32_t* dup = mark_slots<V>(p, lds);
  const uint32_t total = (uint32_t)p.total, first = (uint32_t)p.head[0] % total, count = (uint32_t)p.head[1];
  const uint32_t back = (first + count % total) % total;
  uint32_t fcarry = 0, tcarry = 0;
  for (int b0 = 0; b0 < p.n; b0 += kStepThreads * V) {
    const int b = b0 + tid * V;
    int32_t slot[V], want[V];
    int64_t a[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      slot[v] = b + v < p.n ? p.slots[b + v] : -1;
      want[v] = p.lengths && b + v < p.n ? p.lengths[b + v] : p.chunk;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = (uint32_t)slot[v] < (uint32_t)p.S ? p.appended[slot[v]] : 0;
    StreamPages s[V];
    uint64_t both = 0;  // pages given back and taken: each sum is below 2^32, two in one
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = stream_pages(p, b + v, slot[v], want[v], a[v], dup);
      both += (uint64_t)(uint32_t)s[v].freed << 32 | (uint32_t)s[v].taken;
    }
    // the first page given back of each stream, on its way while the sums meet
    uint32_t r0[V];
    int32_t e0[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      r0[v] = s[v].lo % (uint32_t)p.M;
      e0[v] = s[v].freed > 0 ? p.ring[(int64_t)s[v].slot * p.M + r0[v]] : 0;
    }
    uint64_t all;
    both = block_scan<kStepThreads / 64>(both, sums, all);
    uint32_t f = fcarry + (uint32_t)(both >> 32), t = tcarry + (uint32_t)both;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (s[v].freed > 0) give_back(p, s[v].slot, s[v].freed, r0[v], (back + f) % total, &e0[v]);
      if (of && b + v < p.n) of[b + v] = StepOf{(int32_t)s[v].A, s[v].slot, s[v].len, t};
      if (s[v].slot >= 0) p.appended[s[v].slot] = p.reset ? 0 : (int64_t)s[v].A + s[v].len;
      f += s[v].freed;
      t += s[v].taken;
    }
    fcarry += (uint32_t)(all >> 32);
    tcarry += (uint32_t)all;
  }
  front = first;
  if (tid == 0) {
    p.head[0] = (int32_t)((first + tcarry) % total);
    p.head[1] = (int32_t)(count + fcarry - tcarry);
  }
}

// Rows, and slot map where it is asked for, of a stream by a group of 32 lanes, an entry a lane: ring entry, or the page
// from the queue's front where the entry is one that the step takes.
__device__ static inline void step_rows(const PageK& p, int b, const StepOf s, uint32_t front, int lane) {
  const uint32_t total = (uint32_t)p.total;
  const int P1 = (1 << p.page_shift) - 1;
  const uint32_t hi = ((uint32_t)s.A + P1) >> p.page_shift, hi2 = ((uint32_t)s.A + s.len + P1) >> p.page_shift;
  const int hm = (int)(hi % (uint32_t)p.M), taken = s.slot < 0 ? 0 : (int)(hi2 - hi);
  int32_t* const ring = p.ring + (int64_t)s.slot * p.M;
  // page of the d-th logical page from hi on (-1: the one that A ends in)
  auto page = [&](int d, int r) { return d >= 0 && d < taken ? p.queue[(front + s.at + d) % total] : s.slot < 0 ? -1 : ring[r]; };
  int32_t* const row = p.rows + (int64_t)b * p.rows_stride;
  for (int i = lane; i < 1 + p.M; i += 32) {
    const int r = i - 1, d = r >= hm ? r - hm : r - hm + p.M;
    const int v = i == 0 ? s.A : page(d, r);
    row[i] = v;
    if (i > 0 && d < taken) ring[r] = v;
  }
  if (!p.slot_map) return;
  int32_t* const map = p.slot_map + b * p.map_stride;
  for (int t = lane; t < p.chunk; t += 32) {
    const uint32_t pos = (uint32_t)s.A + t;
    const int d = (int)((pos >> p.page_shift) - hi);
    int r = hm + d;
    r = r < 0 ? r + p.M : r >= p.M ? r - p.M : r;
    map[t] = t < s.len ? (page(d, r) << p.page_shift) + (int)(pos & P1) : -1;
  }
}

// A step of up to kStepOne streams, and a reset, in one launch: bound by its chain of
// round trips to memory (slots, frame counts, rings, queue).
__global__ void __launch_bounds__(kStepThreads) page_step_kernel(const PageK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint64_t sums[kStepThreads / 64];
  __shared__ StepOf of[kStepOne];
  uint32_t front;
  step_scan<1>(p, lds, sums, p.reset ? nullptr : of, front);
  if (p.reset) return;
  __syncthreads();  // every page given back is in the queue
  for (int b = threadIdx.x >> 5; b < p.n; b += kStepThreads / 32) step_rows(p, b, of[b], front, threadIdx.x & 31);
}

// More streams: the part in order by one workgroup, rows and slot map by all of them in a
// second launch.
__global__ void __launch_bounds__(kStepThreads) page_scan_kernel(const PageK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint64_t sums[kStepThreads / 64];
  uint32_t front;
  step_scan<4>(p, lds, sums, p.of, front);
  if (threadIdx.x == 0) *p.front = front;
}
__global__ void __launch_bounds__(256) page_rows_kernel(const PageK p) {
  const int b = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b < p.n) step_rows(p, b, p.of[b], *p.front, threadIdx.x & 31);
}

// Thousands of streams: one CU's scattered reads (0.6 a ns) of their frame counts and
// rings, and its share of the memory's rate, would be the step (16384 streams: 44 us). So a
// workgroup sums what its 256 streams give and take, one workgroup sums the sums and looks
// for equal slots, the pages go back, the rows are written, a launch each.
constexpr int kPartThreads = 256;

__global__ void __launch_bounds__(kPartThreads) page_part_kernel(const PageK p) {
  __shared__ uint64_t sums[kPartThreads / 64];
  const int b = blockIdx.x * kPartThreads + threadIdx.x;
  const int32_t slot = b < p.n ? p.slots[b] : -1, want = p.lengths && b < p.n ? p.lengths[b] : p.chunk;
  const StreamPages s = stream_pages(p, b, slot, want, (uint32_t)slot < (uint32_t)p.S ? p.appended[slot] : 0, nullptr);
  uint64_t all;
  block_scan<kPartThreads / 64>((uint64_t)(uint32_t)s.freed << 32 | (uint32_t)s.taken, sums, all);
  if (b < p.n) {
    p.of[b] = StepOf{(int32_t)s.A, s.slot, s.len, 0};
    p.part[b] = uint2{(uint32_t)s.freed, (uint32_t)s.taken};
  }
  if (threadIdx.x == 0) p.sum[blockIdx.x] = uint2{(uint32_t)(all >> 32), (uint32_t)all};
}

__global__ void __launch_bounds__(kStepThreads) page_sums_kernel(const PageK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint64_t sums[kStepThreads / 64];
  const uint32_t* dup = mark_slots<16>(p, lds);
  uint32_t twice = 0;
  for (int i = threadIdx.x; i < (p.S + 31) >> 5; i += kStepThreads) twice |= dup[i];
  if (__syncthreads_or(twice)) {
    for (int b = threadIdx.x; b < p.n; b += kStepThreads)
      if (named_before(p, b, p.slots[b], dup)) {
        const uint2 s = p.part[b];
        atomicSub(&p.sum[b / kPartThreads].x, s.x);
        atomicSub(&p.sum[b / kPartThreads].y, s.y);
        p.part[b] = uint2{0, 0};
        p.of[b] = StepOf{0, -1, 0, 0};
      }
    __threadfence();
    __syncthreads();
  }
  const uint32_t total = (uint32_t)p.total, first = (uint32_t)p.head[0] % total, count = (uint32_t)p.head[1];
  const int blocks = (p.n + kPartThreads - 1) / kPartThreads;
  uint64_t carry = 0;
  for (int i0 = 0; i0 < blocks; i0 += kStepThreads) {
    const int i = i0 + threadIdx.x;
    const uint2 s = i < blocks ? p.sum[i] : uint2{0, 0};
    uint64_t all;
    const uint64_t at = block_scan<kStepThreads / 64>((uint64_t)s.x << 32 | s.y, sums, all) + carry;
    if (i < blocks) p.sum[i] = uint2{(uint32_t)(at >> 32), (uint32_t)at};
    carry += all;
  }
  if (threadIdx.x == 0) {
    p.front[0] = first;
    p.front[1] = (first + count % total) % total;
    p.head[0] = (int32_t)((first + (uint32_t)carry) % total);
    p.head[1] = (int32_t)(count + (uint32_t)(carry >> 32) - (uint32_t)carry);
  }
}

__global__ void __launch_bounds__(kPartThreads) page_back_kernel(const PageK p) {
  __shared__ uint64_t sums[kPartThreads / 64];
  const int b = blockIdx.x * kPartThreads + threadIdx.x;
  const StepOf s = b < p.n ? p.of[b] : StepOf{0, -1, 0, 0};
  const uint2 part = b < p.n ? p.part[b] : uint2{0, 0}, base = p.sum[blockIdx.x];
  uint64_t all;
  const uint64_t at = block_scan<kPartThreads / 64>((uint64_t)part.x << 32 | part.y, sums, all);
  if (s.slot < 0) return;
  if (part.x) {
    const uint32_t A = (uint32_t)s.A, lo = A > (uint32_t)p.window ? (A - p.window) >> p.page_shift : 0;
    give_back(p, s.slot, part.x, lo % (uint32_t)p.M, (p.front[1] + base.x + (uint32_t)(at >> 32)) % (uint32_t)p.total, nullptr);
  }
  p.of[b].at = base.y + (uint32_t)at;
  p.appended[s.slot] = (int64_t)(uint32_t)s.A + s.len;
}

// ---------------------------------------------------------------------------
// adapter plan
//
// A stable counting sort of the streams by adapter in one workgroup: each wave
// counts a run of the streams (LDS), the counts are summed over waves and adapters,
// and each wave places its run in order, 64 streams at a time, a stream's rank among
// the equal ones of its 64 found with one ballot a bit of the number.  Streams
// without an adapter are bucket G.  Bound by its chain of LDS passes and, for thousands
// of streams, by one CU's instructions: in a graph 128 streams of 2 frames take 5.4 us, 4096 in
// 512 buckets 9.1 (with 14 frames, two launches, 12.6), 16384 22.8.

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kPlanTile = 32;    // rows of a tile
constexpr int kPlanOne = 4096;   // rows of a plan in one launch, streams sorted in LDS

struct PlanK {
  const int32_t* ids;
  int32_t* order;
  int32_t* sorted;
  int4* tiles;
  int32_t B, T, G, max_tiles, bits;
  int2* by;  // {stream, adapter} by position, where rows and tiles are a second launch's
  uint32_t* tab;  // its tables: start [G + 1], tile0 [G + 1]
};

// rows of a tile t: the adapter whose tiles it is among (bisection over their first tiles)
__device__ static inline int4 plan_tile(const PlanK& p, const uint32_t* start, const uint32_t* tile0, int t) {
  if ((uint32_t)t >= tile0[p.G]) return int4{-1, 0, 0, 0};
  int lo = 0, hi = p.G;  // tile0[lo] <= t < tile0[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tile0[mid] <= (uint32_t)t)
      lo = mid;
    else
      hi = mid;
  }
  const int off = (t - (int)tile0[lo]) * kPlanTile;
  return int4{lo, (int)start[lo] * p.T + off, min(kPlanTile, (int)(start[lo + 1] - start[lo]) * p.T - off), 0};
}

__global__ void __launch_bounds__(kPlanThreads) adapter_plan_kernel(const PlanK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint32_t sums[kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int G1 = p.G + 1;
  uint32_t* const hist = lds;                       // [waves][G + 1]
  uint32_t* const start = hist + kPlanWaves * G1;   // [G + 2] first stream of a bucket
  uint32_t* const tile0 = start + G1 + 1;           // [G + 1] first tile of an adapter
  // up to kPlanOne streams: adapter + 1 and stream by position, [B], so that memory gets
  // whole lines
  uint32_t* const placed = tile0 + G1;
  for (int i = tid; i < kPlanWaves * G1; i += kPlanThreads) hist[i] = 0;
  constexpr int U = 4;  // numbers a lane loads at once: 64 U streams a wave and round trip
  auto load_ids = [&](int32_t (&id)[U], int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = p.ids[min(b + 64 * u, p.B - 1)];
  };
  const int run = ((p.B + kPlanWaves - 1) / kPlanWaves + 63) & ~63;
  const int b0 = min(wave * run, p.B), b1 = min(b0 + run, p.B);
  __syncthreads();
  for (int b = b0 + lane; b < b1; b += 64 * U) {
    int32_t id[U];
    load_ids(id, b);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (b + 64 * u < b1) atomicAdd(&hist[wave * G1 + ((uint32_t)id[u] < (uint32_t)p.G ? id[u] : p.G)], 1u);
  }
  __syncthreads();
  // bucket g's streams before each wave's, and before bucket g
  uint32_t carry = 0, tcarry = 0;
  for (int g0 = 0; g0 < G1; g0 += kPlanThreads) {
    const int g = g0 + tid;
    uint32_t h[kPlanWaves], c = 0;  // every wave's at once: one LDS round trip, not 16
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) h[w] = g < G1 ? hist[w * G1 + g] : 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      const uint32_t n = h[w];
      h[w] = c;
      c += n;
    }
    const uint32_t tiles = g < p.G ? (c * p.T + kPlanTile - 1) / kPlanTile : 0;
    uint32_t all, tall;
    const uint32_t s = block_scan<kPlanWaves>(c, sums, all) + carry;
    const uint32_t t = block_scan<kPlanWaves>(tiles, sums, tall) + tcarry;
    if (g < G1) {
      start[g] = s;
      tile0[g] = t;
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) hist[w * G1 + g] = h[w] + s;
    }
    carry += all;
    tcarry += tall;
  }
  __syncthreads();
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int b4 = b0; b4 < b1; b4 += 64 * U) {
    int32_t ids[U];
    load_ids(ids, b4 + lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b4 + 64 * u;
      if (b >= b1) break;
      const bool in = b + lane < b1;
      const int32_t id = in ? ids[u] : -1;
      const bool has = (uint32_t)id < (uint32_t)p.G;
      const int g = has ? id : p.G;
      const uint64_t all = __ballot(in);
      uint32_t lo = (uint32_t)all, up = (uint32_t)(all >> 32);
      for (int i = p.bits; i > 0; --i) {
        const int32_t bit = (int32_t)((uint32_t)g << (32 - i)) >> 31;  // -1 or 0
        const uint64_t m = __ballot(bit);
        lo &= ~((uint32_t)m ^ (uint32_t)bit);
        up &= ~((uint32_t)(m >> 32) ^ (uint32_t)bit);
      }
      const uint64_t same = (uint64_t)up << 32 | lo;
      uint32_t* const h = &hist[wave * G1 + g];
      uint32_t base = 0;
      if (in) base = *h;
      wave_lds_sync();
      if (in && (same >> lane) == 1) *h = base + __popcll(same);  // the last of the equal ones
      wave_lds_sync();
      if (in) {
        const int32_t at = (int32_t)(base + __popcll(same & below));
        if (p.B <= kPlanOne)
          placed[at] = (uint32_t)(has ? id + 1 : 0) << 16 | (uint32_t)(b + lane);
        else
          p.by[at] = int2{b + lane, has ? id : -1};
      }
    }
  }
  __syncthreads();
  if (p.by) {
    if (p.B <= kPlanOne)
      for (int i = tid; i < p.B; i += kPlanThreads) p.by[i] = int2{(int)(placed[i] & 0xffff), (int)(placed[i] >> 16) - 1};
    for (int i = tid; i < 2 * G1; i += kPlanThreads) p.tab[i] = i < G1 ? start[i] : tile0[i - G1];
    return;
  }
  for (int i = tid; i < p.B * p.T; i += kPlanThreads) {
    const int s = i / p.T;
    p.order[i] = (int)(placed[s] & 0xffff) * p.T + (i - s * p.T);
    p.sorted[i] = (int)(placed[s] >> 16) - 1;
  }
  for (int t = tid; t < p.max_tiles; t += kPlanThreads) p.tiles[t] = plan_tile(p, start, tile0, t);
}

// Many rows: theirs and the tiles in a second launch, by all CUs (57344 rows in 512 buckets:
// one workgroup stores 0.5 MB in 50 us).
__global__ void __launch_bounds__(256) adapter_rows_kernel(const PlanK p) {
  const int i = blockIdx.x * 256 + threadIdx.x;  // B T and max_tiles: below 2^24
  if (i < p.B * p.T) {
    const int s = i / p.T;
    const int2 v = p.by[s];
    p.order[i] = v.x * p.T + (i - s * p.T);
    p.sorted[i] = v.y;
  }
  if (i < p.max_tiles) p.tiles[i] = plan_tile(p, p.tab, p.tab + p.G + 1, i);
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
  if (a->batch > PK_PAGE_STEP_MAX_SLOTS)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d streams (built: up to %d)", what, a->batch, PK_PAGE_STEP_MAX_SLOTS);
  if (a->batch == 0) return PK_OK;
  if (!a->queue || !a->head || !a->appended || !a->ring || !a->slots)
    return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (!a->reset) {
    if (!a->rows) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
    if (a->rows_stride < 1 + M || (a->slot_map && a->slot_map_stride < a->chunk))
      return fail(PK_ERR_INVALID, "%s: need rows_stride >= %d and slot_map_stride >= %d", what, 1 + M, a->chunk);
  }
  const bool two = !a->reset && a->batch > kStepOne;
  if (two && (!a->workspace || !aligned16(a->workspace)))
    return fail(PK_ERR_INVALID, "%s: workspace must be non-NULL and 16-byte aligned for %d streams", what, a->batch);
  PageK k{};
  k.queue = a->queue;
  k.head = a->head;
  k.appended = a->appended;
  k.ring = a->ring;
  k.slots = a->slots;
  k.lengths = a->reset ? nullptr : a->lengths;  // a reset's may be any address
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
  if (two) {
    k.of = static_cast<StepOf*>(a->workspace);
    k.front = reinterpret_cast<uint32_t*>(k.of + k.n);
    k.part = reinterpret_cast<uint2*>(k.of + k.n + 1);
    k.sum = k.part + k.n;
  }
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const size_t bits = (size_t)((k.S + 31) / 32) * 8;
  if (!two) {
    hipLaunchKernelGGL(page_step_kernel, dim3(1), dim3(kStepThreads), bits, s, k);
    return check_launch(what);
  }
  const dim3 all((unsigned)((k.n + kPartThreads - 1) / kPartThreads));
  if (k.n <= kStepTwo) {
    hipLaunchKernelGGL(page_scan_kernel, dim3(1), dim3(kStepThreads), bits, s, k);
  } else {
    hipLaunchKernelGGL(page_part_kernel, all, dim3(kPartThreads), 0, s, k);
    hipLaunchKernelGGL(page_sums_kernel, dim3(1), dim3(kStepThreads), bits, s, k);
    hipLaunchKernelGGL(page_back_kernel, all, dim3(kPartThreads), 0, s, k);
  }
  hipLaunchKernelGGL(page_rows_kernel, dim3((unsigned)((k.n + 7) / 8)), dim3(256), 0, s, k);
  return check_launch(what);
}

int adapter_plan(const pk_adapter_plan_args* a, hipStream_t s) {
  const char* what = "pk_adapter_plan";
  // a projection's rows are at least 128 bytes and its tensors below 2^31
  if (a->batch < 0 || a->frames <= 0 || a->num_adapters <= 0 || (int64_t)a->batch * a->frames >= (int64_t{1} << 24))
    return fail(PK_ERR_INVALID, "%s: need batch >= 0, frames and num_adapters > 0, and fewer than 2^24 rows (got %d, %d, %d)", what,
                a->batch, a->frames, a->num_adapters);
  if (a->num_adapters > PK_ADAPTER_MAX)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d adapters (built: up to %d)", what, a->num_adapters, PK_ADAPTER_MAX);
  const int64_t need = pk_adapter_plan_tiles(a->batch, a->frames, a->num_adapters);
  if (a->max_tiles < need || a->max_tiles >= (1 << 24))
    return fail(PK_ERR_INVALID, "%s: %d tiles, needs %d and takes fewer than 2^24", what, a->max_tiles, (int)need);
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
  if (pk_adapter_plan_workspace_bytes(k.B, k.T, k.G) > 0) {
    if (!a->workspace || !aligned16(a->workspace))
      return fail(PK_ERR_INVALID, "%s: workspace must be non-NULL and 16-byte aligned for %d rows", what, k.B * k.T);
    k.by = static_cast<int2*>(a->workspace);
    k.tab = reinterpret_cast<uint32_t*>(k.by + k.B);
  }
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const size_t lds = sizeof(uint32_t) * ((size_t)kPlanWaves * (k.G + 1) + 2 * (k.G + 2) + (k.B <= kPlanOne ? k.B : 0));  // below 64 KB
  hipLaunchKernelGGL(adapter_plan_kernel, dim3(1), dim3(kPlanThreads), lds, s, k);
  int rc = check_launch(what);
  if (rc != PK_OK || !k.by) return rc;
  const int rows = k.B * k.T > k.max_tiles ? k.B * k.T : k.max_tiles;
  hipLaunchKernelGGL(adapter_rows_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, s, k);
  return check_launch(what);
}

}  // namespace
}  // namespace pk

extern "C" int64_t pk_page_step_workspace_bytes(int32_t batch) {
  if (batch <= pk::kStepOne) return 0;
  const int64_t blocks = ((int64_t)batch + pk::kPartThreads - 1) / pk::kPartThreads;
  return ((int64_t)batch + 1) * sizeof(pk::StepOf) + (batch > pk::kStepTwo ? (batch + blocks) * (int64_t)sizeof(uint2) : 0);
}

extern "C" int pk_page_step(const pk_page_step_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_page_step: args is NULL");
  return pk::page_step(args, static_cast<hipStream_t>(stream));
}

extern "C" int pk_adapter_plan_tiles(int32_t batch, int32_t frames, int32_t num_adapters) {
  if (batch <= 0 || frames <= 0 || num_adapters <= 0) return 0;
  return (int)((int64_t)batch * frames / pk::kPlanTile + (num_adapters < batch ? num_adapters : batch));
}

extern "C" int64_t pk_adapter_plan_workspace_bytes(int32_t batch, int32_t frames, int32_t num_adapters) {
  if (batch <= 0 || frames <= 0 || num_adapters <= 0 || (int64_t)batch * frames <= pk::kPlanOne) return 0;
  return (int64_t)batch * sizeof(int2) + 2 * ((int64_t)num_adapters + 1) * sizeof(uint32_t);
}

extern "C" int pk_adapter_plan(const pk_adapter_plan_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_adapter_plan: args is NULL");
  return pk::adapter_plan(args, static_cast<hipStream_t>(stream));
}
