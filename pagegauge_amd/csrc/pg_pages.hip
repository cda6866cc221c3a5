// Pages of a pool: copied between places, counted, handed out, and moved together.
//
// A pool is any number of planes (codes, scales, exact pages, of one layer or several)
// that share their page ids, and an int32 count of users per page.  Counts are
// changed by atomic additions of whole numbers, and pages are handed out and moved in
// the order of their ids, so every result is the same from run to run.
#include "pg_common.h"

#include <algorithm>

namespace pg {
namespace {

// plain vectors: structs of them, not yet loaded, would go through LDS
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kPlanesPerLaunch = 32;

// ---- copies -------------------------------------------------------------

struct CopyPlane {
  uint8_t* base;
  int64_t page_stride, row_stride;   // bytes
  uint32_t page_units;               // vectors of a page
  int32_t shift;                     // log2(page_units), or -1
  int32_t log_bytes;                 // of a vector: 4 (16 bytes) to 0
  uint32_t first_block;              // of this plane in the grid
  uint32_t row_blocks;               // blocks of one of its rows
};

struct CopyArgs {
  CopyPlane planes[kPlanesPerLaunch];
  const int32_t* source;
  const int32_t* target;
  uint32_t moves;
  int32_t pages;
  int planes_used;
};

constexpr int kCopyInFlight = 4;     // vectors of a thread
constexpr uint32_t kCopyBlock = kThreads * kCopyInFlight;

template <typename T>
__device__ __forceinline__ void copy_block(const CopyArgs& a, const CopyPlane& p, uint8_t* row, uint32_t first) {
  T value[kCopyInFlight];
  int64_t to[kCopyInFlight];
#pragma unroll
  for (int i = 0; i < kCopyInFlight; ++i) {
    const uint64_t at = static_cast<uint64_t>(first) * kCopyBlock + i * kThreads + threadIdx.x;
    const uint64_t move = p.shift >= 0 ? at >> p.shift : at / p.page_units;
    to[i] = -1;
    if (move < a.moves) {
      const int64_t unit = static_cast<int64_t>(at - move * p.page_units) * sizeof(T);
      const int32_t source = a.source[move], target = a.target[move];
      if (source >= 0 && source < a.pages && target >= 0 && target < a.pages) {
        to[i] = target * p.page_stride + unit;
        value[i] = *reinterpret_cast<const T*>(row + source * p.page_stride + unit);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kCopyInFlight; ++i)
    if (to[i] >= 0) *reinterpret_cast<T*>(row + to[i]) = value[i];
}

// A plane's row (one layer) is copied as one sequence of the moves' pages, in blocks of
// 1024 vectors of 16 bytes (or what the page's size and place allow).  Bound by HBM: 540
// exact pages of K and V in 8 layers, 566 MB read and written, 95 to 101 us (5.6 to 6.0 TB/s;
// a copy of 1 GiB reaches 5.1), 8 pages 3.8 us; a list with empty entries costs their
// workgroups (4096 moves of an INT8 pool in 8192 entries, 268 MB, 67 us: 4.0 TB/s).
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a) {
  int plane = 0;
  while (plane + 1 < a.planes_used && blockIdx.x >= a.planes[plane + 1].first_block) ++plane;
  const CopyPlane& p = a.planes[plane];
  const uint32_t block = blockIdx.x - p.first_block;
  const uint32_t row_index = block / p.row_blocks, first = block % p.row_blocks;
  uint8_t* row = p.base + row_index * p.row_stride;
  switch (p.log_bytes) {
    case 4: return copy_block<v4u>(a, p, row, first);
    case 3: return copy_block<v2u>(a, p, row, first);
    case 2: return copy_block<uint32_t>(a, p, row, first);
    case 1: return copy_block<uint16_t>(a, p, row, first);
    default: return copy_block<uint8_t>(a, p, row, first);
  }
}

// ---- counts -------------------------------------------------------------

// A thread per id: a trip to memory and an atomic (8192 ids 3 to 5 us).
__global__ __launch_bounds__(kThreads) void adjust_kernel(int32_t* refs, int32_t pages, const int32_t* ids,
                                                          int64_t count, int32_t by) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= count) return;
  const int32_t id = ids[i];
  if (id < 0 || id >= pages) return;
  if (by > 0) {
    // Past int32 the count would be that of a free page: it is put to the largest one and
    // stays there.  The last to touch a count that passed it is one that puts it there: the
    // first addition after that passes it again.
    if (atomicAdd(refs + id, by) > INT32_MAX - by) atomicExch(refs + id, INT32_MAX);
    return;
  }
  // never below zero: a page that nobody uses stays free
  int32_t seen = refs[id];
  while (seen > 0 && seen < INT32_MAX) {
    const int32_t old = atomicCAS(refs + id, seen, max(seen + by, 0));
    if (old == seen) break;
    seen = old;
  }
}

__global__ __launch_bounds__(kThreads) void rewrite_kernel(const int32_t* ids, const int32_t* remap, int32_t pages,
                                                           int64_t count, int32_t* out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= count) return;
  const int32_t id = ids[i];
  out[i] = id < 0 || id >= pages ? id : remap[id];
}

// ---- scans over the counts ----------------------------------------------

// One workgroup goes over the pool in stretches of 16384 pages, 16 neighbouring ones
// per thread, so that an order by thread is an order by page.
constexpr int kScanThreads = 1024;
constexpr int kScanPages = 16;
constexpr int kStretch = kScanThreads * kScanPages;

// Bits of the thread's pages first .. first + 15 that are in use; 0 past the end.
__device__ __forceinline__ uint32_t live_bits(const int32_t* refs, int64_t first, int32_t pages) {
  uint32_t bits = 0;
  if (first + kScanPages <= pages) {
    int4 x[kScanPages / 4];
#pragma unroll
    for (int i = 0; i < kScanPages / 4; ++i) x[i] = reinterpret_cast<const int4*>(refs + first)[i];
#pragma unroll
    for (int i = 0; i < kScanPages / 4; ++i)
      bits |= (x[i].x > 0 ? 1u : 0u) << (4 * i) | (x[i].y > 0 ? 2u : 0u) << (4 * i) |
              (x[i].z > 0 ? 4u : 0u) << (4 * i) | (x[i].w > 0 ? 8u : 0u) << (4 * i);
  } else {
    for (int i = 0; i < kScanPages; ++i)
      if (first + i < pages && refs[first + i] > 0) bits |= 1u << i;
  }
  return bits;
}

// Sum over the workgroup, and in ``before`` that of the threads in front.
__device__ __forceinline__ int block_scan(int value, int& before, int* wave_sums) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int x = value;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int y = __shfl_up(x, d, kWave);
    if (lane >= d) x += y;
  }
  if (lane == kWave - 1) wave_sums[wave] = x;
  __syncthreads();
  int front = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kScanThreads / kWave; ++w) {
    const int s = wave_sums[w];
    front += w < wave ? s : 0;
    all += s;
  }
  __syncthreads();
  before = front + x - value;
  return all;
}

// The lowest free pages in order, stretch by stretch until there are enough.  Bound by the trips of
// one workgroup: 64 pages of 16384 half in use 3.4 us and of 300000 4.9, all free ones (so
// the whole pool) 8.7 and 149.
__global__ __launch_bounds__(kScanThreads) void take_kernel(int32_t* refs, int32_t pages, int32_t* out,
                                                            int64_t count) {
  __shared__ int wave_sums[kScanThreads / kWave];
  int64_t found = 0;
  for (int64_t stretch = 0; stretch < pages && found < count; stretch += kStretch) {
    const int64_t first = stretch + threadIdx.x * kScanPages;
    const int held = static_cast<int>(max(min(pages - first, static_cast<int64_t>(kScanPages)), int64_t{0}));
    uint32_t free = ~live_bits(refs, first, pages) & ((1u << held) - 1);
    int before;
    const int all = block_scan(__popc(free), before, wave_sums);
    for (int64_t at = found + before; free && at < count; ++at, free &= free - 1) {
      const int32_t page = static_cast<int32_t>(first + __ffs(free) - 1);
      out[at] = page;
      refs[page] = 1;
    }
    found += all;
  }
  for (int64_t i = found + threadIdx.x; i < count; i += kScanThreads) out[i] = -1;
}

// The pages in use, ``live`` of them, are to fill the pool's front: the i-th lowest page
// at or past ``live`` that is in use goes to the i-th lowest free one below it, the
// fewest moves there are.  No page is both a source and a target.  Bound by the trips of one
// workgroup, which larger pools take one stretch after the other: 1021 pages 5.9 us, 16384
// 10.3, 131072 71, 300000 169 (the first two with a scan for each list and entries of remap
// stored one by one 14.4 and 7.2; over masks of 64 neighbouring pages, more than the scalar
// registers hold, 18.2 and 9.8 to 12.2).
__global__ __launch_bounds__(kScanThreads) void stage_kernel(const int32_t* refs, int32_t pages, int32_t* source,
                                                             int32_t* target, int32_t* remap, int32_t* live_out) {
  __shared__ int wave_sums[kScanThreads / kWave];
  int live = 0, before;
  uint32_t used = 0;
  for (int64_t stretch = 0; stretch < pages; stretch += kStretch) {
    used = live_bits(refs, stretch + threadIdx.x * kScanPages, pages);
    live += block_scan(__popc(used), before, wave_sums);
  }
  if (threadIdx.x == 0) *live_out = live;
  int holes = 0, movers = 0;
  for (int64_t stretch = 0; stretch < pages; stretch += kStretch) {
    const int64_t first = stretch + threadIdx.x * kScanPages;
    const int below = static_cast<int>(max(min(live - first, static_cast<int64_t>(kScanPages)), int64_t{0}));
    if (pages > kStretch) used = live_bits(refs, first, pages);       // of one stretch they are in hand
    uint32_t hole = ~used & ((1u << below) - 1);
    uint32_t mover = used & ~((1u << below) - 1);
    // both counts of a stretch fit 16 bits; pages below ``live`` are pages of the pool
    const int all = block_scan(__popc(hole) << 16 | __popc(mover), before, wave_sums);
    for (int at = holes + (before >> 16); hole; ++at, hole &= hole - 1)
      target[at] = static_cast<int32_t>(first + __ffs(hole) - 1);
    for (int at = movers + (before & 0xffff), left = mover; left; ++at, left &= left - 1)
      source[at] = static_cast<int32_t>(first + __ffs(left) - 1);
    // movers' entries follow below
    const uint32_t stays = used & ~mover;
    auto entry = [&](int i) { return stays >> i & 1 ? static_cast<int32_t>(first + i) : -1; };
    if (first + kScanPages <= pages) {
#pragma unroll
      for (int i = 0; i < kScanPages; i += 4)
        *reinterpret_cast<int4*>(remap + first + i) = make_int4(entry(i), entry(i + 1), entry(i + 2), entry(i + 3));
    } else {
      for (int i = 0; first + i < pages; ++i) remap[first + i] = entry(i);
    }
    holes += all >> 16;
    movers += all & 0xffff;
  }
  __syncthreads();
  const int half = pages / 2;
  for (int i = threadIdx.x; i < half; i += kScanThreads) {
    if (i < movers) {
      remap[source[i]] = target[i];
    } else {
      source[i] = -1;
      target[i] = -1;
    }
  }
}

__global__ __launch_bounds__(kThreads) void commit_kernel(int32_t* refs, int32_t pages, const int32_t* source,
                                                          const int32_t* target, int32_t moves) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= moves) return;
  const int32_t from = source[i], to = target[i];
  if (from < 0 || from >= pages || to < 0 || to >= pages) return;
  if (refs[from] <= 0) return;       // moved already, or given back since
  refs[to] = refs[from];
  refs[from] = 0;
}

int log2_of(uint64_t x) { return x && !(x & (x - 1)) ? __builtin_ctzll(x) : -1; }

unsigned blocks_of(int64_t count, int64_t per_block) { return static_cast<unsigned>((count + per_block - 1) / per_block); }

// Workgroups of a launch: the grid counts its threads in 32 bits.
constexpr int64_t kMaxBlocks = (int64_t{1} << 32) / kThreads - 1;

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_copy_pages(const pg_page_plane_t* host_planes, int32_t planes, int64_t pages,
                                 const int32_t* source, const int32_t* target, int64_t moves, void* stream) {
  clear_error();
  if (planes < 0 || (planes && !host_planes)) return fail(PG_ERROR_INVALID_ARGUMENT, "null planes");
  if (pages < 0 || pages > INT32_MAX || moves < 0 || moves > INT32_MAX)
    return fail(PG_ERROR_INVALID_ARGUMENT, "pages and moves must lie in [0, 2^31)");
  if (moves && (!source || !target)) return fail(PG_ERROR_INVALID_ARGUMENT, "null page ids");
  for (int32_t i = 0; i < planes; ++i) {
    const pg_page_plane_t& p = host_planes[i];
    if (!p.base || p.page_bytes <= 0 || p.rows < 0 || p.page_bytes > INT32_MAX)
      return fail(PG_ERROR_INVALID_ARGUMENT, "a plane needs an address, rows >= 0 and pages of 1 to 2^31 - 1 bytes");
    if (p.page_stride < p.page_bytes)
      return fail(PG_ERROR_INVALID_ARGUMENT, "pages of a plane must not overlap");
  }
  if (!moves || !pages) return PG_OK;
  CopyArgs a{};
  a.source = source;
  a.target = target;
  a.moves = static_cast<uint32_t>(moves);
  a.pages = static_cast<int32_t>(pages);
  int64_t blocks = 0;
  auto launch = [&]() -> int32_t {
    if (!a.planes_used) return PG_OK;
    hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                       as_stream(stream), a);
    a.planes_used = 0;
    blocks = 0;
    return check_launch("copy_pages");
  };
  for (int32_t i = 0; i < planes; ++i) {
    const pg_page_plane_t& p = host_planes[i];
    CopyPlane c{};
    c.page_stride = p.page_stride;
    c.row_stride = p.row_stride;
    const uint64_t places = reinterpret_cast<uintptr_t>(p.base) | static_cast<uint64_t>(p.page_bytes) |
                            static_cast<uint64_t>(p.page_stride) |
                            (p.rows > 1 ? static_cast<uint64_t>(p.row_stride) : 0);
    c.log_bytes = std::min(4, __builtin_ctzll(places));
    c.page_units = static_cast<uint32_t>(p.page_bytes >> c.log_bytes);
    c.shift = log2_of(c.page_units);
    const int64_t row_blocks = (moves * c.page_units + kCopyBlock - 1) / kCopyBlock;
    if (row_blocks > kMaxBlocks) return fail(PG_ERROR_UNSUPPORTED, "too many bytes for one copy");
    c.row_blocks = static_cast<uint32_t>(row_blocks);
    // rows in as many launches as the grid's limit asks for
    for (int64_t row = 0; row < p.rows;) {
      if (a.planes_used == kPlanesPerLaunch || blocks + row_blocks > kMaxBlocks)
        if (int32_t rc = launch()) return rc;
      const int64_t rows = std::min(p.rows - row, (kMaxBlocks - blocks) / row_blocks);
      c.base = static_cast<uint8_t*>(p.base) + row * p.row_stride;
      c.first_block = static_cast<uint32_t>(blocks);
      a.planes[a.planes_used++] = c;
      blocks += rows * row_blocks;
      row += rows;
    }
  }
  return launch();
}

static int32_t check_pool(const void* refs, int64_t pages) {
  if (pages < 0 || pages > INT32_MAX) return fail(PG_ERROR_INVALID_ARGUMENT, "pages must lie in [0, 2^31)");
  if (pages && !refs) return fail(PG_ERROR_INVALID_ARGUMENT, "null pool");
  if (reinterpret_cast<uintptr_t>(refs) % 16) return fail(PG_ERROR_INVALID_ARGUMENT, "counts must be 16-byte aligned");
  return PG_OK;
}

extern "C" int32_t pg_pool_adjust(int32_t* refs, int64_t pages, const int32_t* ids, int64_t count, int32_t by,
                                  void* stream) {
  clear_error();
  if (int32_t rc = check_pool(refs, pages)) return rc;
  if (count < 0 || count > kMaxBlocks * kThreads) return fail(PG_ERROR_INVALID_ARGUMENT, "too many ids");
  if (count && !ids) return fail(PG_ERROR_INVALID_ARGUMENT, "null page ids");
  if (!count || !pages || !by) return PG_OK;
  hipLaunchKernelGGL(adjust_kernel, dim3(blocks_of(count, kThreads)), dim3(kThreads), 0, as_stream(stream), refs,
                     static_cast<int32_t>(pages), ids, count, by);
  return check_launch("pool_adjust");
}

extern "C" int32_t pg_pool_take(int32_t* refs, int64_t pages, int32_t* out, int64_t count, void* stream) {
  clear_error();
  if (int32_t rc = check_pool(refs, pages)) return rc;
  if (count < 0) return fail(PG_ERROR_INVALID_ARGUMENT, "the count must be nonnegative");
  if (!count) return PG_OK;
  if (!out) return fail(PG_ERROR_INVALID_ARGUMENT, "null page ids");
  hipLaunchKernelGGL(take_kernel, dim3(1), dim3(kScanThreads), 0, as_stream(stream), refs,
                     static_cast<int32_t>(pages), out, count);
  return check_launch("pool_take");
}

extern "C" int32_t pg_pool_stage_compaction(const int32_t* refs, int64_t pages, int32_t* source, int32_t* target,
                                            int32_t* remap, int32_t* live, void* stream) {
  clear_error();
  if (int32_t rc = check_pool(refs, pages)) return rc;
  if (reinterpret_cast<uintptr_t>(remap) % 16) return fail(PG_ERROR_INVALID_ARGUMENT, "remap must be 16-byte aligned");
  if (!live || (pages && !remap) || (pages > 1 && (!source || !target)))
    return fail(PG_ERROR_INVALID_ARGUMENT, "null output of a compaction");
  hipLaunchKernelGGL(stage_kernel, dim3(1), dim3(kScanThreads), 0, as_stream(stream), refs,
                     static_cast<int32_t>(pages), source, target, remap, live);
  return check_launch("pool_stage_compaction");
}

extern "C" int32_t pg_pool_commit_compaction(int32_t* refs, int64_t pages, const int32_t* source,
                                             const int32_t* target, int64_t moves, void* stream) {
  clear_error();
  if (int32_t rc = check_pool(refs, pages)) return rc;
  if (moves < 0 || moves > pages) return fail(PG_ERROR_INVALID_ARGUMENT, "more moves than pages");
  if (moves && (!source || !target)) return fail(PG_ERROR_INVALID_ARGUMENT, "null page ids");
  if (!moves) return PG_OK;
  hipLaunchKernelGGL(commit_kernel, dim3(blocks_of(moves, kThreads)), dim3(kThreads), 0, as_stream(stream), refs,
                     static_cast<int32_t>(pages), source, target, static_cast<int32_t>(moves));
  return check_launch("pool_commit_compaction");
}

extern "C" int32_t pg_rewrite_ids(const int32_t* ids, const int32_t* remap, int64_t pages, int64_t count,
                                  int32_t* out, void* stream) {
  clear_error();
  if (pages < 0 || pages > INT32_MAX || count < 0 || count > kMaxBlocks * kThreads)
    return fail(PG_ERROR_INVALID_ARGUMENT, "pages and ids must lie in [0, 2^31)");
  if (!count) return PG_OK;
  if (!ids || !out || (pages && !remap)) return fail(PG_ERROR_INVALID_ARGUMENT, "null page ids");
  hipLaunchKernelGGL(rewrite_kernel, dim3(blocks_of(count, kThreads)), dim3(kThreads), 0, as_stream(stream), ids,
                     remap, static_cast<int32_t>(pages), count, out);
  return check_launch("rewrite_ids");
}
