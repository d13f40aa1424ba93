// gfx950 page work of a device page pool beyond a step's (tables_kernels.hip): streams
// continued in other slots, the live pages moved together, and the copies of K and V that
// both ask for.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "pk_common.h"
#include "pk_device.h"
#include "pk_scan.h"

namespace pk {

// ---------------------------------------------------------------------------
// fork
//
// A slot of A frames holds the logical pages lo(A) .. hi(A) (tables_kernels.hip). All
// destinations give their pages back, then all pages are taken: with a pool of num_slots * M
// pages or more the queue cannot run dry, since after the call too no slot holds more than M.
// What a pair gives and takes is known from the frame counts, so two prefix sums over the
// pairs place every page.

struct ForkOf {
  int32_t src, dst;       // dst -1: absent
  uint32_t lo, freed;     // the destination's first logical page, and how many
  uint32_t slo, taken;    // the source's
  uint32_t back, at;      // pages given back and taken by the pairs before
};

struct ForkK {
  int32_t* queue;
  int32_t* head;
  int64_t* appended;
  int32_t* ring;
  const int32_t* src;
  const int32_t* dst;
  int2* pairs;
  int32_t* count;
  int32_t n, S, total, M, page_shift, window;
  ForkOf* of;       // [n]
  uint32_t* front;  // {first entry, entry behind the last, pages taken}
};

constexpr int kForkThreads = 1024;

// first logical page held and their number, of a slot of `a` frames
__device__ static inline void held_pages(const ForkK& p, int64_t a, uint32_t& lo, uint32_t& n) {
  const uint32_t A = (uint32_t)min(max(a, (int64_t)0), (int64_t)0x7fffffff), P1 = (1u << p.page_shift) - 1u;
  lo = A > (uint32_t)p.window ? (A - p.window) >> p.page_shift : 0;
  n = (A >> p.page_shift) + ((A & P1) != 0) - lo;
}

// The pairs' part that has to be in order, by one workgroup: who is absent, the sums over the
// pairs, the queue's new ends.
__device__ static inline void fork_scan(const ForkK& p, uint32_t* lds, uint64_t* sums, ForkOf* of, uint32_t* front) {
  const int tid = threadIdx.x, words = (p.S + 31) >> 5;
  uint32_t* const named = lds;            // bits of the sources
  uint32_t* const seen = named + words;   // of the destinations
  uint32_t* const twice = seen + words;   // of those named more than once
  for (int i = tid; i < 3 * words; i += kForkThreads) lds[i] = 0;
  __syncthreads();
  for (int b = tid; b < p.n; b += kForkThreads) {
    const int32_t s = p.src[b], d = p.dst[b];
    if ((uint32_t)s < (uint32_t)p.S) atomicOr(&named[s >> 5], 1u << (s & 31));
    if ((uint32_t)d < (uint32_t)p.S) {
      const uint32_t bit = 1u << (d & 31);
      if (atomicOr(&seen[d >> 5], bit) & bit) atomicOr(&twice[d >> 5], bit);
    }
  }
  __syncthreads();
  const uint32_t total = (uint32_t)p.total, first = (uint32_t)p.head[0] % total, entries = (uint32_t)p.head[1];
  uint32_t fcarry = 0, tcarry = 0;
  for (int b0 = 0; b0 < p.n; b0 += kForkThreads) {
    const int b = b0 + tid;
    ForkOf f{};
    f.src = b < p.n ? p.src[b] : -1;
    f.dst = b < p.n ? p.dst[b] : -1;
    bool in = (uint32_t)f.src < (uint32_t)p.S && (uint32_t)f.dst < (uint32_t)p.S;
    if (in && (named[f.dst >> 5] >> (f.dst & 31) & 1)) in = false;
    // the first of equal destinations has the pair (rare: a search of the pairs before)
    if (in && (twice[f.dst >> 5] >> (f.dst & 31) & 1))
      for (int j = 0; j < b && in; j += 8)
#pragma unroll
        for (int u = 0; u < 8; ++u) in &= p.dst[min(j + u, b - 1)] != f.dst;
    if (in) {
      held_pages(p, p.appended[f.dst], f.lo, f.freed);
      held_pages(p, p.appended[f.src], f.slo, f.taken);
    } else {
      f.dst = -1;
    }
    uint64_t all;
    const uint64_t at = block_scan<kForkThreads / 64>((uint64_t)f.freed << 32 | f.taken, sums, all);
    f.back = fcarry + (uint32_t)(at >> 32);
    f.at = tcarry + (uint32_t)at;
    if (b < p.n) of[b] = f;
    fcarry += (uint32_t)(all >> 32);
    tcarry += (uint32_t)all;
  }
  __syncthreads();  // every frame count and the queue's ends are read
  if (tid == 0) {
    front[0] = first;
    front[1] = (first + entries % total) % total;
    front[2] = tcarry;
    p.head[0] = (int32_t)((first + tcarry) % total);
    p.head[1] = (int32_t)(entries + fcarry - tcarry);
    *p.count = (int32_t)tcarry;
  }
}

// the j-th page of a destination back to the queue
__device__ static inline void fork_back(const ForkK& p, const ForkOf& f, uint32_t j, const uint32_t* front) {
  if (f.dst < 0 || j >= f.freed) return;
  const uint32_t total = (uint32_t)p.total, at = (front[1] + f.back % total + j) % total;
  p.queue[at] = p.ring[(int64_t)f.dst * p.M + (f.lo + j) % (uint32_t)p.M];
}

// Ring entry j of a destination: the page for the source's, or none; the pair's moves.
__device__ static inline void fork_entry(const ForkK& p, const ForkOf& f, uint32_t j, const uint32_t* front) {
  if (f.dst < 0) return;
  const uint32_t total = (uint32_t)p.total, M = (uint32_t)p.M, r = (f.slo + j) % M;
  int32_t page = -1;
  if (j < f.taken) {
    page = p.queue[(front[0] + f.at % total + j) % total];
    p.pairs[f.at + j] = int2{p.ring[(int64_t)f.src * M + r], page};
  }
  p.ring[(int64_t)f.dst * M + r] = page;
  if (j == 0) p.appended[f.dst] = p.appended[f.src];
}

// A few pairs in one launch: bound by its chain of round trips (4 pairs of 32 slots: 4.3 us, 48 of 230: 4.7).
constexpr int kForkOne = 256, kForkOneEntries = 8192;  // pairs, and their ring entries
__global__ void __launch_bounds__(kForkThreads) page_fork_kernel(const ForkK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint64_t sums[kForkThreads / 64];
  __shared__ ForkOf of[kForkOne];
  __shared__ uint32_t front[3];
  fork_scan(p, lds, sums, of, front);
  __syncthreads();
  const int entries = p.n * p.M;
  for (int i = threadIdx.x; i < entries; i += kForkThreads) fork_back(p, of[i / p.M], (uint32_t)(i % p.M), front);
  __syncthreads();  // every page given back is in the queue
  for (int i = threadIdx.x; i < entries; i += kForkThreads) {
    fork_entry(p, of[i / p.M], (uint32_t)(i % p.M), front);
    if (i >= (int)front[2]) p.pairs[i] = int2{-1, -1};
  }
}

// More: the part in order by one workgroup, pages back and pages taken by all of them.
__global__ void __launch_bounds__(kForkThreads) fork_scan_kernel(const ForkK p) {
  extern __shared__ uint32_t lds[];
  __shared__ uint64_t sums[kForkThreads / 64];
  fork_scan(p, lds, sums, p.of, p.front);
}
__global__ void __launch_bounds__(256) fork_back_kernel(const ForkK p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < p.n * p.M) fork_back(p, p.of[i / p.M], (uint32_t)(i % p.M), p.front);
}
__global__ void __launch_bounds__(256) fork_rows_kernel(const ForkK p) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.n * p.M) return;
  fork_entry(p, p.of[i / p.M], (uint32_t)(i % p.M), p.front);
  if (i >= (int)p.front[2]) p.pairs[i] = int2{-1, -1};
}

// ---------------------------------------------------------------------------
// compaction
//
// A bit a page says whether a slot holds it, `before` how many held pages come before each
// word of bits. With N held pages in all, the held page p >= N of rank r among those takes
// the place of the free page of rank r below N: as many are held from N on as are free below.

struct CompactK {
  int32_t* queue;
  int32_t* head;
  int32_t* ring;
  int2* pairs;
  int32_t* count;
  int32_t total, words, capacity;
  int64_t entries;  // num_slots * M
  uint32_t* bits;    // [words]
  uint32_t* before;  // [words + 1], the last: N
};

constexpr int kCompactThreads = 1024;

// held pages below p, p <= total
__device__ static inline uint32_t held_below(const uint32_t* bits, const uint32_t* before, uint32_t p) {
  const uint32_t rest = p & 31;
  return before[p >> 5] + (rest ? __popc(bits[p >> 5] & ((1u << rest) - 1u)) : 0u);
}

__device__ static inline void compact_mark(const CompactK& p, uint32_t* bits, int64_t i) {
  const uint32_t page = (uint32_t)p.ring[i];
  if (page < (uint32_t)p.total) atomicOr(&bits[page >> 5], 1u << (page & 31));
}

__device__ static inline void compact_sum(const CompactK& p, const uint32_t* bits, uint32_t* before, uint32_t* sums) {
  uint32_t carry = 0;
  for (int w0 = 0; w0 < p.words; w0 += kCompactThreads) {
    const int w = w0 + threadIdx.x;
    uint32_t all;
    const uint32_t at = block_scan<kCompactThreads / 64>(w < p.words ? (uint32_t)__popc(bits[w]) : 0u, sums, all);
    if (w < p.words) before[w] = carry + at;
    carry += all;
  }
  if (threadIdx.x == 0) {
    before[p.words] = carry;
    p.head[0] = 0;
    p.head[1] = p.total - (int32_t)carry;
  }
}

// page i: its end of a move, its place in the queue, an unused move
__device__ static inline void compact_page(const CompactK& p, const uint32_t* bits, const uint32_t* before, uint32_t i) {
  const uint32_t N = before[p.words], below = held_below(bits, before, i), kept = held_below(bits, before, N), moves = N - kept;
  const bool held = bits[i >> 5] >> (i & 31) & 1;
  if (i < N && !held) p.pairs[i - below].y = (int32_t)i;
  if (i >= N && held) p.pairs[below - kept].x = (int32_t)i;
  if (i < (uint32_t)p.total - N) p.queue[i] = (int32_t)(N + i);
  if (i >= moves && i < (uint32_t)p.capacity) p.pairs[i] = int2{-1, -1};
  if (i == 0) *p.count = (int32_t)moves;
}

__device__ static inline void compact_entry(const CompactK& p, const uint32_t* bits, const uint32_t* before, int64_t i) {
  const uint32_t page = (uint32_t)p.ring[i], N = before[p.words];
  if (page >= N && page < (uint32_t)p.total) p.ring[i] = p.pairs[held_below(bits, before, page) - held_below(bits, before, N)].y;
}

// Small pools in one launch, bits in LDS (230 slots of 7 entries: 4.7 us).
constexpr int kCompactOne = 32768;  // pages
__global__ void __launch_bounds__(kCompactThreads) page_compact_kernel(const CompactK p) {
  __shared__ uint32_t bits[kCompactOne / 32], before[kCompactOne / 32 + 1], sums[kCompactThreads / 64];
  for (int w = threadIdx.x; w < p.words; w += kCompactThreads) bits[w] = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < p.entries; i += kCompactThreads) compact_mark(p, bits, i);
  __syncthreads();
  compact_sum(p, bits, before, sums);
  __syncthreads();
  for (int i = threadIdx.x; i < p.total; i += kCompactThreads) compact_page(p, bits, before, (uint32_t)i);
  __syncthreads();
  for (int64_t i = threadIdx.x; i < p.entries; i += kCompactThreads) compact_entry(p, bits, before, i);
}

// Large ones by all workgroups, bits in the workspace.
__global__ void __launch_bounds__(256) compact_clear_kernel(const CompactK p) {
  const int w = blockIdx.x * 256 + threadIdx.x;
  if (w < p.words) p.bits[w] = 0;
}
__global__ void __launch_bounds__(256) compact_mark_kernel(const CompactK p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < p.entries) compact_mark(p, p.bits, i);
}
__global__ void __launch_bounds__(kCompactThreads) compact_sum_kernel(const CompactK p) {
  __shared__ uint32_t sums[kCompactThreads / 64];
  compact_sum(p, p.bits, p.before, sums);
}
__global__ void __launch_bounds__(256) compact_pages_kernel(const CompactK p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i < (uint32_t)p.total) compact_page(p, p.bits, p.before, i);
}
__global__ void __launch_bounds__(256) compact_rings_kernel(const CompactK p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < p.entries) compact_entry(p, p.bits, p.before, i);
}

// ---------------------------------------------------------------------------
// the copies
//
// A page of a layer is contiguous, so a move is a plain copy, layer by layer in K and V,
// in units of 256 x kMoveChunks 16-byte pieces, past the caches (nothing in a call is read twice:
// 250 pages of 24 layers and 32 KB, 0.8 GB read and written, 161 us so, 166 through them, where a large
// copy takes 152). The number of moves is known to the GPU alone: workgroups stride over the units.

struct MoveK {
  u32x4* k;
  u32x4* v;
  const int2* pairs;
  const int32_t* count;
  int32_t capacity, layers, num_pages, units;  // units of a page
  uint32_t chunks;   // 16-byte pieces of a page
};

constexpr int kMoveChunks = 4;
__global__ void __launch_bounds__(256) kv_move_kernel(const MoveK p) {
  const uint32_t n = (uint32_t)min(max(*p.count, 0), p.capacity);
  const uint32_t per = (uint32_t)p.layers * 2 * p.units;  // units of a pair, below 2^31
  const uint64_t all = (uint64_t)n * per;
  for (uint64_t i = blockIdx.x; i < all; i += gridDim.x) {
    const uint32_t m = (uint32_t)(i / per);
    uint32_t r = (uint32_t)(i - (uint64_t)m * per);
    const uint32_t unit = r % (uint32_t)p.units;
    r /= (uint32_t)p.units;
    const int2 pair = p.pairs[m];
    if ((uint32_t)pair.x >= (uint32_t)p.num_pages || (uint32_t)pair.y >= (uint32_t)p.num_pages) continue;
    u32x4* const pool = (r & 1 ? p.v : p.k) + (int64_t)(r >> 1) * p.num_pages * p.chunks;
    const u32x4* const from = pool + (int64_t)pair.x * p.chunks;
    u32x4* const to = pool + (int64_t)pair.y * p.chunks;
    const uint32_t c = unit * (256 * kMoveChunks) + threadIdx.x;
    u32x4 x[kMoveChunks];
#pragma unroll
    for (int u = 0; u < kMoveChunks; ++u)
      if (c + 256 * u < p.chunks) x[u] = __builtin_nontemporal_load(from + c + 256 * u);
#pragma unroll
    for (int u = 0; u < kMoveChunks; ++u)
      if (c + 256 * u < p.chunks) __builtin_nontemporal_store(x[u], to + c + 256 * u);
  }
}

namespace {

int page_fork(const pk_page_fork_args* a, hipStream_t s) {
  const char* what = "pk_page_fork";
  const int ps = log2_of(a->page_size);
  if (ps < 0) return fail(PK_ERR_INVALID, "%s: page_size %d is not a power of two", what, a->page_size);
  if (a->left < 0 || a->chunk <= 0 || a->num_slots <= 0 || a->num_pages <= 0 || a->batch < 0 ||
      (int64_t)a->left + a->chunk + a->page_size >= (int64_t{1} << 31))
    return fail(PK_ERR_INVALID, "%s: need left >= 0, chunk, num_slots and num_pages > 0, batch >= 0 (got %d, %d, %d, %d, %d)", what,
                a->left, a->chunk, a->num_slots, a->num_pages, a->batch);
  const int32_t M = (a->left + a->chunk + a->page_size - 2) / a->page_size + 1;
  if ((int64_t)a->num_pages < (int64_t)a->num_slots * M || a->num_pages >= (1 << 30))
    return fail(PK_ERR_INVALID, "%s: %d pages cannot hold %d slots of %d pages each (or are 2^30 or more)", what, a->num_pages, a->num_slots, M);
  if (a->num_slots > PK_PAGE_STEP_MAX_SLOTS)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d slots (built: up to %d)", what, a->num_slots, PK_PAGE_STEP_MAX_SLOTS);
  if (a->batch > a->num_slots) return fail(PK_ERR_INVALID, "%s: %d pairs for %d slots", what, a->batch, a->num_slots);
  if (!a->queue || !a->head || !a->appended || !a->ring || !a->count || (a->batch > 0 && (!a->src || !a->dst || !a->pairs)))
    return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (reinterpret_cast<uintptr_t>(a->pairs) & 7u) return fail(PK_ERR_INVALID, "%s: pairs must be 8-byte aligned", what);
  const bool one = pk_page_fork_workspace_bytes(a->batch, M) == 0;
  if (!one && (!a->workspace || !aligned16(a->workspace)))
    return fail(PK_ERR_INVALID, "%s: workspace must be non-NULL and 16-byte aligned for %d pairs", what, a->batch);
  ForkK k{};
  k.queue = a->queue;
  k.head = a->head;
  k.appended = a->appended;
  k.ring = a->ring;
  k.src = a->src;
  k.dst = a->dst;
  k.pairs = reinterpret_cast<int2*>(a->pairs);
  k.count = a->count;
  k.n = a->batch;
  k.S = a->num_slots;
  k.total = a->num_pages;
  k.M = M;
  k.page_shift = ps;
  k.window = a->left + a->chunk;
  if (!one) {
    k.of = static_cast<ForkOf*>(a->workspace);
    k.front = reinterpret_cast<uint32_t*>(k.of + k.n);
  }
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const size_t bits = (size_t)((k.S + 31) / 32) * 12;  // 48 KB at most
  if (one) {
    hipLaunchKernelGGL(page_fork_kernel, dim3(1), dim3(kForkThreads), bits, s, k);
    return check_launch(what);
  }
  const dim3 all((unsigned)(((int64_t)k.n * M + 255) / 256));
  hipLaunchKernelGGL(fork_scan_kernel, dim3(1), dim3(kForkThreads), bits, s, k);
  hipLaunchKernelGGL(fork_back_kernel, all, dim3(256), 0, s, k);
  hipLaunchKernelGGL(fork_rows_kernel, all, dim3(256), 0, s, k);
  return check_launch(what);
}

int page_compact(const pk_page_compact_args* a, hipStream_t s) {
  const char* what = "pk_page_compact";
  if (a->num_slots <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->num_pages >= (1 << 30))
    return fail(PK_ERR_INVALID, "%s: need num_slots and max_pages > 0 and 0 < num_pages < 2^30 (got %d, %d, %d)", what, a->num_slots, a->max_pages,
                a->num_pages);
  const int64_t entries = (int64_t)a->num_slots * a->max_pages;
  if (entries > a->num_pages) return fail(PK_ERR_INVALID, "%s: %d pages cannot hold %d slots of %d pages each", what, a->num_pages, a->num_slots, a->max_pages);
  const int64_t need = entries < a->num_pages / 2 ? entries : a->num_pages / 2;
  if (a->capacity < need) return fail(PK_ERR_INVALID, "%s: room for %d moves, needs %d", what, a->capacity, (int)need);
  if (!a->queue || !a->head || !a->ring || !a->count || (a->capacity > 0 && !a->pairs))
    return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (reinterpret_cast<uintptr_t>(a->pairs) & 7u) return fail(PK_ERR_INVALID, "%s: pairs must be 8-byte aligned", what);
  CompactK k{};
  k.queue = a->queue;
  k.head = a->head;
  k.ring = a->ring;
  k.pairs = reinterpret_cast<int2*>(a->pairs);
  k.count = a->count;
  k.total = a->num_pages;
  k.words = (a->num_pages + 31) / 32;
  k.capacity = a->capacity < a->num_pages ? a->capacity : a->num_pages;
  k.entries = entries;
  const bool one = pk_page_compact_workspace_bytes(entries, a->num_pages) == 0;
  if (!one) {
    if (!a->workspace || !aligned16(a->workspace))
      return fail(PK_ERR_INVALID, "%s: workspace must be non-NULL and 16-byte aligned for %d pages", what, a->num_pages);
    k.bits = static_cast<uint32_t*>(a->workspace);
    k.before = k.bits + k.words;
  }
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  if (one) {
    hipLaunchKernelGGL(page_compact_kernel, dim3(1), dim3(kCompactThreads), 0, s, k);
    return check_launch(what);
  }
  auto grid = [](int64_t n) { return dim3((unsigned)((n + 255) / 256)); };
  hipLaunchKernelGGL(compact_clear_kernel, grid(k.words), dim3(256), 0, s, k);
  hipLaunchKernelGGL(compact_mark_kernel, grid(entries), dim3(256), 0, s, k);
  hipLaunchKernelGGL(compact_sum_kernel, dim3(1), dim3(kCompactThreads), 0, s, k);
  hipLaunchKernelGGL(compact_pages_kernel, grid(k.total), dim3(256), 0, s, k);
  hipLaunchKernelGGL(compact_rings_kernel, grid(entries), dim3(256), 0, s, k);
  return check_launch(what);
}

int kv_move_pages(const pk_kv_move_pages_args* a, hipStream_t s) {
  const char* what = "pk_kv_move_pages";
  if (a->dtype != PK_DTYPE_F32 && a->dtype != PK_DTYPE_F16 && a->dtype != PK_DTYPE_BF16)
    return fail(PK_ERR_INVALID, "%s: unknown dtype %d", what, a->dtype);
  const pk_paged_layout& L = a->pages;
  if (L.num_layers <= 0 || L.num_pages <= 0 || L.page_size <= 0 || L.d_model <= 0)
    return fail(PK_ERR_INVALID, "%s: need layers, pages, page_size and d_model > 0", what);
  const int64_t bytes = (int64_t)L.page_size * L.d_model * (a->dtype == PK_DTYPE_F32 ? 4 : 2);
  if (bytes % 16 != 0 || bytes >= (int64_t{1} << 31))
    return fail(PK_ERR_INVALID, "%s: pages of %lld bytes are not multiples of 16 below 2^31", what, (long long)bytes);
  if (a->capacity < 0) return fail(PK_ERR_INVALID, "%s: capacity < 0", what);
  if (a->capacity == 0) return PK_OK;
  if (!L.k_pool || !L.v_pool || !a->pairs || !a->count) return fail(PK_ERR_INVALID, "%s: a tensor pointer is NULL", what);
  if (!aligned16(L.k_pool) || !aligned16(L.v_pool) || (reinterpret_cast<uintptr_t>(a->pairs) & 7u))
    return fail(PK_ERR_INVALID, "%s: pools must be 16-byte aligned and pairs 8-byte", what);
  MoveK k{};
  k.k = static_cast<u32x4*>(L.k_pool);
  k.v = static_cast<u32x4*>(L.v_pool);
  k.pairs = reinterpret_cast<const int2*>(a->pairs);
  k.count = a->count;
  k.capacity = a->capacity;
  k.layers = L.num_layers;
  k.num_pages = L.num_pages;
  k.chunks = (uint32_t)(bytes / 16);
  k.units = (int32_t)((k.chunks + 256 * kMoveChunks - 1) / (256 * kMoveChunks));
  const int64_t per = (int64_t)k.layers * 2 * k.units;
  if (per >= (int64_t{1} << 31)) return fail(PK_ERR_INVALID, "%s: a page of all layers is past 2^31 units", what);
  DeviceGuard dg(a->device);
  if (!dg.ok) return fail(PK_ERR_HIP, "%s: cannot select device %d", what, a->device);
  const int64_t most = (int64_t)cu_count() * 8, units = per * a->capacity;
  hipLaunchKernelGGL(kv_move_kernel, dim3((unsigned)(units < most ? units : most)), dim3(256), 0, s, k);
  return check_launch(what);
}

}  // namespace
}  // namespace pk

extern "C" {

int64_t pk_page_fork_workspace_bytes(int32_t batch, int32_t max_pages) {
  if (batch <= pk::kForkOne && (int64_t)batch * max_pages <= pk::kForkOneEntries) return 0;
  return ((int64_t)batch + 1) * (int64_t)sizeof(pk::ForkOf);
}

int pk_page_fork(const pk_page_fork_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_page_fork: args is NULL");
  return pk::page_fork(args, static_cast<hipStream_t>(stream));
}

int64_t pk_page_compact_workspace_bytes(int64_t ring_entries, int32_t num_pages) {
  if (num_pages <= pk::kCompactOne && ring_entries <= pk::kCompactOne) return 0;
  return (2 * (((int64_t)num_pages + 31) / 32) + 1) * (int64_t)sizeof(uint32_t);
}

int pk_page_compact(const pk_page_compact_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_page_compact: args is NULL");
  return pk::page_compact(args, static_cast<hipStream_t>(stream));
}

int pk_kv_move_pages(const pk_kv_move_pages_args* args, void* stream) {
  pk::clear_error();
  if (!args) return pk::fail(PK_ERR_INVALID, "pk_kv_move_pages: args is NULL");
  return pk::kv_move_pages(args, static_cast<hipStream_t>(stream));
}

}  // extern "C"
