// Attention over a part of a request's pages, picked per KV head by bounds of their keys:
// the bounds, the scores that they give, the choice, and the attention over it.
//
// Bounds are the least and the largest K code of each channel of a (page, KV head).  For a
// query row q, the largest product that a key between them (lo <= hi) could have is
//   sum_d max(q_d hi_d, q_d lo_d) = sum_d q+_d hi_d + q-_d lo_d,   q+ = max(q, 0), q- = min(q, 0),
// a product of 256 terms, and with q in whole steps of a power of two, one of 8-bit integers
// on the matrix cores: exact, so that the choice does not depend on an order of additions.
#include "pg_page_attention.h"

namespace pg {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v2i16 __attribute__((ext_vector_type(2)));

// ---- bounds -------------------------------------------------------------

constexpr int kBoundsThreads = 256;
constexpr int kPieces = kHeadDim / 16;       // threads of a (page, head): 16 channels each

struct BoundsArgs {
  const uint8_t* codes;
  uint8_t* bounds;               // [pages, Hkv, 2, 128]
  const int32_t* page_ids;       // or null: page i
  const int32_t* lengths;        // or null: 16
  int64_t units;                 // listed pages * heads * kPieces
  int32_t pool_pages;
  uint32_t heads;
};

__device__ __forceinline__ v2i16 as_pair(uint32_t x) { return __builtin_bit_cast(v2i16, x); }

// A thread takes 16 channels of a page's 16 tokens, all requested at once; neighbouring
// threads take neighbouring channels and heads, so a wave reads whole token rows.  Signed
// bytes are compared as the high bytes of 16-bit halves: the odd ones where they are, the
// even ones a byte further up.  Bound by the reads: 8191 pages of 8 heads, 151 MB, in 22.8 us
// where they are still in the Infinity Cache and 32 where not (4.6 TB/s); 32 pages 3.3 us.
__global__ __launch_bounds__(kBoundsThreads) void key_bounds_kernel(BoundsArgs a) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kBoundsThreads + threadIdx.x;
  if (unit >= a.units) return;
  const uint32_t row_units = a.heads * kPieces;
  const int64_t i = unit / row_units;
  const uint32_t piece = static_cast<uint32_t>(unit - i * row_units);
  const int32_t page = a.page_ids ? a.page_ids[i] : static_cast<int32_t>(i);
  if (page < 0 || page >= a.pool_pages) return;
  const int length = a.lengths ? max(min(a.lengths[i], kPageSize), 0) : kPageSize;
  const uint32_t row_bytes = a.heads * kHeadDim;
  const uint8_t* from = a.codes + static_cast<int64_t>(page) * kPageSize * row_bytes + piece * 16;
  v4u x[kPageSize];
#pragma unroll
  for (int t = 0; t < kPageSize; ++t)    // rows past the page's tokens are its last one again
    x[t] = *reinterpret_cast<const v4u*>(from + min(t, max(length - 1, 0)) * row_bytes);
  v2i16 low[8], high[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    low[d] = as_pair(0x7f7f7f7fu);
    high[d] = as_pair(0x80808080u);
  }
#pragma unroll
  for (int t = 0; t < kPageSize; ++t) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const v2i16 odd = as_pair(x[t][d]);
      const v2i16 even = odd << 8;
      low[d] = __builtin_elementwise_min(low[d], odd);
      high[d] = __builtin_elementwise_max(high[d], odd);
      low[4 + d] = __builtin_elementwise_min(low[4 + d], even);
      high[4 + d] = __builtin_elementwise_max(high[4 + d], even);
    }
  }
  v4u least, most;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    // bytes 1 and 3 of the odd halves, and of the even ones, back in order
    least[d] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, low[d]), __builtin_bit_cast(uint32_t, low[4 + d]), 0x07030501u);
    most[d] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, high[d]), __builtin_bit_cast(uint32_t, high[4 + d]), 0x07030501u);
  }
  if (length == 0) {
    least = v4u{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
    most = v4u{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
  }
  uint8_t* to = a.bounds + (static_cast<int64_t>(page) * a.heads + piece / kPieces) * 2 * kHeadDim + piece % kPieces * 16;
  *reinterpret_cast<v4u*>(to) = least;
  *reinterpret_cast<v4u*>(to + kHeadDim) = most;
}

// ---- scores -------------------------------------------------------------

struct SelectArgs {
  const uint16_t* query;
  int64_t query_batch_stride;
  const uint8_t* bounds;
  const uint16_t* key_scale;       // [pages, Hkv]
  const int32_t* indices;
  const int32_t* indptr;           // [B + 1]
  float* scores;                   // [Hkv, pages] of each request, one after the other
  int32_t* selected;               // [B, Hkv, take]
  int take, first, last;
  int num_kv_heads, group, wave_groups;
};

constexpr int kScoreThreads = 256;
constexpr int kScorePages = 16;      // rows of an MFMA
constexpr int kMostGroups = 8;       // of so many pages, per wave: two page ids a lane

// Sixteen pages at a time are the rows of v_mfma_i32_16x16x64_i8 and the KV head's query
// heads its columns; 4 products take the 128 lower bounds and the 128 upper ones.  Page ids
// and scales are requested once per wave, a group's bounds while the one before is scored.
// Bound by the reads of bounds: 65536 pages of 8 heads, 134 MB, 26 to 28 us where the Infinity
// Cache still has some, 34 where not (3.9 TB/s; the same with a page's heads side by side).
__global__ __launch_bounds__(kScoreThreads) void page_scores_kernel(SelectArgs a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int n = lane & 15, kg = lane >> 4;
  const int kv = blockIdx.y, request = blockIdx.z, hkv = a.num_kv_heads;
  const int begin = a.indptr[request], pages = a.indptr[request + 1] - begin;
  if (pages <= a.take) return;       // all of them are taken
  const int first = (blockIdx.x * (kScoreThreads / kWave) + wave) * a.wave_groups * kScorePages;
  if (first >= pages) return;

  // lane l has the page ids and scales of the wave's pages l and 64 + l
  const int last = min(first + a.wave_groups * kScorePages, pages) - 1;
  int ids[2];
  float scales[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) ids[i] = a.indices[begin + min(first + 64 * i + lane, last)];

  // the head's query in steps of a power of two, at most 127 of them
  v4i below[2], above[2];
  float unit;
  {
    const uint16_t* row = a.query + request * a.query_batch_stride +
                          static_cast<int64_t>(kv * a.group + n % a.group) * kHeadDim;
    uint32_t bits[2][8];
    uint32_t most = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const v4u x = *reinterpret_cast<const v4u*>(row + 64 * w + 16 * kg + 8 * d);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bits[w][4 * d + e] = x[e];
          most = max(most, max(x[e] & 0x7fffu, x[e] >> 16 & 0x7fffu));
        }
      }
    most = max(most, __shfl_xor(most, 16, kWave));
    most = max(most, __shfl_xor(most, 32, kWave));
    // largest = f 2^x, f in [0.5, 1): steps of 2^(x - 7)
    const float largest = half_bits_to_float(static_cast<uint16_t>(most));
    int x = 0;
    if (most) x = static_cast<int>(__float_as_uint(largest) >> 23) - 126;
    const float up = __uint_as_float(static_cast<uint32_t>(7 - x + 127) << 23);
    // a row with an infinity or NaN has no scores
    unit = most >= 0x7c00u ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(x - 7 + 127) << 23);
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        uint32_t minus = 0, plus = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t half = static_cast<uint16_t>(bits[w][2 * d + e / 2] >> 16 * (e & 1));
          const float steps = most >= 0x7c00u ? 0.0f : rintf(half_bits_to_float(half) * up);
          const int whole = static_cast<int>(fminf(fmaxf(steps, -127.0f), 127.0f));
          minus |= static_cast<uint32_t>(min(whole, 0) & 0xff) << 8 * e;
          plus |= static_cast<uint32_t>(max(whole, 0)) << 8 * e;
        }
        below[w][d] = static_cast<int>(minus);
        above[w][d] = static_cast<int>(plus);
      }
  }

  const uint8_t* bounds = a.bounds + kv * 2 * kHeadDim + 16 * kg;
  auto load = [&](int g, v4i (&x)[4]) {
    const int64_t page = max(__shfl(g < 4 ? ids[0] : ids[1], kScorePages * (g & 3) + n, kWave), 0);
    const uint8_t* from = bounds + page * hkv * 2 * kHeadDim;
#pragma unroll
    for (int w = 0; w < 4; ++w) x[w] = *reinterpret_cast<const v4i*>(from + 64 * w);
  };
  float* scores = a.scores + static_cast<int64_t>(begin - a.indptr[0]) * hkv + static_cast<int64_t>(kv) * pages;
  auto compute = [&](int g, const v4i (&x)[4]) {
    v4i sum = {0, 0, 0, 0};
    sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[0], below[0], sum, 0, 0, 0);
    sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[1], below[1], sum, 0, 0, 0);
    sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[2], above[0], sum, 0, 0, 0);
    sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[3], above[1], sum, 0, 0, 0);
    float best[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // |sum| < 2^21: one rounding, of its product with the FP16 scale
      const float scale = __shfl(g < 4 ? scales[0] : scales[1], kScorePages * (g & 3) + 4 * kg + r, kWave);
      best[r] = row16_max(fmaxf(static_cast<float>(sum[r]) * scale * unit, kNoScore));
    }
    const int position = first + g * kScorePages + 4 * kg + n;
    if (n < 4 && position <= last) scores[position] = n == 0 ? best[0] : n == 1 ? best[1] : n == 2 ? best[2] : best[3];
  };
  const int groups = (last - first) / kScorePages + 1;
  v4i x[2][4];
  load(0, x[0]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // an entry below 0 is no page and has no score: the pool's first one is read in its place
    const float scale = half_bits_to_float(a.key_scale[static_cast<int64_t>(max(ids[i], 0)) * hkv + kv]);
    scales[i] = ids[i] < 0 ? __uint_as_float(0x7fc00000u) : scale;
  }
  for (int g = 0; g < groups; g += 2) {
    if (g + 1 < groups) load(g + 1, x[1]);
    compute(g, x[0]);
    if (g + 1 >= groups) break;
    if (g + 2 < groups) load(g + 2, x[0]);
    compute(g + 1, x[1]);
  }
}

// ---- the choice ---------------------------------------------------------

constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / kWave;
constexpr int kBins = 2 * kPickThreads;
constexpr int kListed = 1024;        // scores near the last one taken that are compared one by one

// Whole numbers in the order of the scores, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float score) {
  const uint32_t bits = __float_as_uint(score == 0.0f ? 0.0f : score);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float score_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// One workgroup per (KV head, request): the last score that is taken, then everything above
// it and the lowest positions at it, in order.  A histogram over 2048 equal parts of the
// scores' range leaves a few to be ranked one by one, or where very many are alike, to
// further histograms over their bits.  Up to kHeld scores stay in a thread's registers;
// with kHeld = 0 they are read again each time.  Scores are no NaN; here NaN stands for a
// page that is taken anyway.
//
// Bound by its chain of steps between barriers: 8 workgroups of 2048 pages 5.9 us, 64 of 8192
// 9.2 (with scores as ordered whole numbers throughout 11.1, as three histograms over their
// bits, read from memory each time, 17.4: scores share their leading bits, and additions
// to one bin wait for each other).
template <int kHeld>
__global__ __launch_bounds__(kPickThreads) void pick_pages_kernel(SelectArgs a) {
  __shared__ uint32_t bins[kBins];
  __shared__ float list[kListed];
  __shared__ uint32_t counts[kHeld > 0 ? kHeld * kPickWaves : kPickWaves];
  __shared__ uint32_t wave_sums[kPickWaves];
  __shared__ float wave_low[kPickWaves], wave_high[kPickWaves];
  __shared__ uint32_t found[3], listed;
  __shared__ float found_score;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int kv = blockIdx.x, request = blockIdx.y;
  const int begin = a.indptr[request], pages = a.indptr[request + 1] - begin;
  int32_t* out = a.selected + (static_cast<int64_t>(request) * a.num_kv_heads + kv) * a.take;
  if (pages <= a.take) {
    for (int i = tid; i < a.take; i += kPickThreads) out[i] = i < pages ? i : -1;
    return;
  }
  const float* scores = a.scores + static_cast<int64_t>(begin - a.indptr[0]) * a.num_kv_heads +
                        static_cast<int64_t>(kv) * pages;
  const float anyway = __uint_as_float(0x7fc00000u);
  auto score_at = [&](int i) { return i < a.first || i >= pages - a.last ? anyway : scores[i]; };
  float held[kHeld > 0 ? kHeld : 1];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = tid + j * kPickThreads;
    held[j] = i < pages ? score_at(i) : anyway;
  }
  auto each_score = [&](auto&& body) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (held[j] == held[j]) body(held[j]);
    } else {
      for (int i = tid; i < pages; i += kPickThreads) {
        const float s = score_at(i);
        if (s == s) body(s);
      }
    }
  };

  // the bin of ``bins`` in which the wanted-th largest key falls, its rank there, and how
  // many keys the bin has
  auto find_bin = [&](uint32_t wanted) {
    const int top = kBins - 2 - 2 * tid;
    const uint32_t upper = bins[top + 1], lower = bins[top];
    uint32_t x = upper + lower;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t y = __shfl_up(x, d, kWave);
      if (lane >= d) x += y;
    }
    if (lane == kWave - 1) wave_sums[wave] = x;
    __syncthreads();
    uint32_t above = x - upper - lower;
    for (int w = 0; w < wave; ++w) above += wave_sums[w];
    if (above < wanted && wanted <= above + upper + lower) {
      const bool in_upper = wanted <= above + upper;
      found[0] = in_upper ? top + 1 : top;
      found[1] = wanted - (in_upper ? above : above + upper);
      found[2] = in_upper ? upper : lower;
    }
    __syncthreads();
  };
  auto clear_bins = [&]() {
    bins[tid] = 0;
    bins[tid + kPickThreads] = 0;
  };

  uint32_t wanted = a.take - a.first - a.last;       // rank of the last score taken, from the top
  float last_score = anyway;                         // none
  if (wanted > 0) {
    float low = -kNoScore, high = kNoScore;
    each_score([&](float s) {
      if (fabsf(s) < -kNoScore) {
        low = fminf(low, s);
        high = fmaxf(high, s);
      }
    });
    low = -wave_max(-low);
    high = wave_max(high);
    if (lane == 0) {
      wave_low[wave] = low;
      wave_high[wave] = high;
    }
    clear_bins();
    if (tid == 0) listed = 0;
    __syncthreads();
    low = -row16_max(-wave_low[lane % kPickWaves]);
    high = row16_max(wave_high[lane % kPickWaves]);
    // rounded alike for all, and never falling as the score rises
    const float per_bin = (kBins - 1) / fmaxf(high - low, 0x1p-100f);
    auto bin_of = [&](float s) {
      return static_cast<uint32_t>(fminf(fmaxf((s - low) * per_bin, 0.0f), static_cast<float>(kBins - 1)));
    };
    each_score([&](float s) { atomicAdd(&bins[bin_of(s)], 1u); });
    __syncthreads();
    find_bin(wanted);
    const uint32_t bin = found[0];
    wanted = found[1];
    if (found[2] <= kListed) {
      each_score([&](float s) {
        if (bin_of(s) == bin) list[atomicAdd(&listed, 1u)] = s;
      });
      __syncthreads();
      const uint32_t count = listed;
      if (static_cast<uint32_t>(tid) < count) {
        const float mine = list[tid];
        uint32_t larger = 0, equal = 0;
        for (uint32_t i = 0; i < count; ++i) {
          larger += list[i] > mine;
          equal += list[i] == mine;
        }
        if (larger < wanted && wanted <= larger + equal) {
          found_score = mine;
          found[1] = wanted - larger;
        }
      }
      __syncthreads();
      last_score = found_score;
      wanted = found[1];
    } else {
      uint32_t key = 0;
      int shift = 32;
#pragma unroll 1
      for (int step = 0; step < 3; ++step) {         // 11 bits, then 11, then 10
        const int width = step < 2 ? 11 : 10, before = shift;
        shift -= width;
        __syncthreads();
        clear_bins();
        __syncthreads();
        each_score([&](float s) {
          const uint32_t at = order_key(s);
          if (bin_of(s) == bin && (before == 32 || at >> before == key >> before))
            atomicAdd(&bins[at >> shift & ((1u << width) - 1)], 1u);
        });
        __syncthreads();
        find_bin(wanted);
        key |= found[0] << shift;
        wanted = found[1];
      }
      last_score = score_of(key);
    }
  }

  // larger scores and the pages taken anyway, and of the equal ones the first ``wanted``
  auto classes = [&](int i, float s, uint64_t& larger, uint64_t& equal) {
    larger = __builtin_amdgcn_ballot_w64(i < pages && (s != s || s > last_score));
    equal = __builtin_amdgcn_ballot_w64(i < pages && s == last_score);
  };
  const uint64_t lanes_below = (1ull << lane) - 1;
  auto write = [&](int i, uint64_t larger, uint64_t equal, uint32_t larger_before, uint32_t equal_before) {
    larger_before += __popcll(larger & lanes_below);
    equal_before += __popcll(equal & lanes_below);
    if ((larger >> lane & 1) || ((equal >> lane & 1) && equal_before < wanted))
      out[larger_before + min(equal_before, wanted)] = i;
  };
  if constexpr (kHeld > 0) {
    // counts of (stretch, wave) in the order of positions, 16 bits each
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      uint64_t larger, equal;
      classes(tid + j * kPickThreads, held[j], larger, equal);
      if (lane == 0)
        counts[j * kPickWaves + wave] = static_cast<uint32_t>(__popcll(larger)) | static_cast<uint32_t>(__popcll(equal)) << 16;
    }
    __syncthreads();
    constexpr int kCounts = kHeld * kPickWaves;
    constexpr int kEach = (kCounts + kWave - 1) / kWave;
    if (wave == 0) {
      uint32_t mine[kEach], sum = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int at = lane * kEach + e;
        mine[e] = at < kCounts ? counts[at] : 0;
        sum += mine[e];
      }
      uint32_t x = sum;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const uint32_t y = __shfl_up(x, d, kWave);
        if (lane >= d) x += y;
      }
      x -= sum;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int at = lane * kEach + e;
        if (at < kCounts) counts[at] = x;
        x += mine[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      uint64_t larger, equal;
      classes(tid + j * kPickThreads, held[j], larger, equal);
      const uint32_t front = counts[j * kPickWaves + wave];
      write(tid + j * kPickThreads, larger, equal, front & 0xffff, front >> 16);
    }
  } else {
    uint32_t larger_so_far = 0, equal_so_far = 0;
    for (int first = 0; first < pages; first += kPickThreads) {
      const int i = first + tid;
      uint64_t larger, equal;
      classes(i, i < pages ? score_at(i) : anyway, larger, equal);
      if (lane == 0)
        wave_sums[wave] = static_cast<uint32_t>(__popcll(larger)) | static_cast<uint32_t>(__popcll(equal)) << 16;
      __syncthreads();
      uint32_t front = 0, all = 0;
      for (int w = 0; w < kPickWaves; ++w) {
        if (w < wave) front += wave_sums[w];
        all += wave_sums[w];
      }
      write(i, larger, equal, larger_so_far + (front & 0xffff), equal_so_far + (front >> 16));
      larger_so_far += all & 0xffff;
      equal_so_far += all >> 16;
      __syncthreads();
    }
  }
}

template <bool kWide>
__global__ __launch_bounds__(kAttentionThreads, 2) void selected_attention_kernel(PageAttentionArgs a) {
  __shared__ NarrowMeeting<kWide> meet;
  // KV heads vary fastest: with 8 of them each XCD reads one head's lines
  const SegmentItem it = a.items[blockIdx.x / a.num_kv_heads];
  page_attention<true, true, kWide>(a, it, blockIdx.x % a.num_kv_heads, meet);
}

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_sparse_key_bounds(const void* key_codes, void* bounds, int64_t pool_pages,
                                        const int32_t* page_ids, const int32_t* lengths, int64_t count,
                                        int32_t kv_heads, void* stream) {
  clear_error();
  if (kv_heads <= 0 || kv_heads > 1024) return fail(PG_ERROR_INVALID_ARGUMENT, "KV heads must lie in [1, 1024]");
  if (pool_pages < 0 || pool_pages > INT32_MAX || count < 0 || count > INT32_MAX)
    return fail(PG_ERROR_INVALID_ARGUMENT, "pages must lie in [0, 2^31)");
  if (!page_ids && count > pool_pages) return fail(PG_ERROR_INVALID_ARGUMENT, "more pages than the pool holds");
  if (!count || !pool_pages) return PG_OK;
  if (!key_codes || !bounds) return fail(PG_ERROR_INVALID_ARGUMENT, "null pages");
  if (reinterpret_cast<uintptr_t>(key_codes) % 16 || reinterpret_cast<uintptr_t>(bounds) % 16)
    return fail(PG_ERROR_INVALID_ARGUMENT, "codes and bounds must be 16-byte aligned");
  BoundsArgs a{};
  a.codes = static_cast<const uint8_t*>(key_codes);
  a.bounds = static_cast<uint8_t*>(bounds);
  a.page_ids = page_ids;
  a.lengths = lengths;
  a.units = count * kv_heads * kPieces;
  a.pool_pages = static_cast<int32_t>(pool_pages);
  a.heads = static_cast<uint32_t>(kv_heads);
  const int64_t blocks = (a.units + kBoundsThreads - 1) / kBoundsThreads;
  if (blocks > UINT32_MAX / kBoundsThreads) return fail(PG_ERROR_UNSUPPORTED, "too many pages for one launch");
  hipLaunchKernelGGL(key_bounds_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kBoundsThreads), 0,
                     as_stream(stream), a);
  return check_launch("key_bounds");
}

extern "C" int32_t pg_sparse_plan(const int32_t* host_indptr, const int32_t* host_tail_indptr, int32_t batch_size,
                                  int32_t num_qo_heads, int32_t num_kv_heads, int32_t selected_pages,
                                  int32_t first_pages, int32_t last_pages, int32_t num_cus, void* workspace,
                                  int64_t workspace_bytes, pg_segment_plan_t* plan, void* stream) {
  clear_error();
  if (selected_pages <= 0) return fail(PG_ERROR_INVALID_ARGUMENT, "at least one page must be selected");
  if (first_pages < 0 || last_pages < 0 || first_pages > selected_pages - last_pages)
    return fail(PG_ERROR_INVALID_ARGUMENT, "first and last pages must fit the selection");
  if (batch_size > 65535) return fail(PG_ERROR_UNSUPPORTED, "at most 65535 requests");
  if (int32_t rc = plan_into({nullptr, nullptr, 0, host_indptr, host_tail_indptr, batch_size, num_qo_heads,
                              num_kv_heads, PG_KV_INT8, selected_pages, num_cus}, workspace, workspace_bytes,
                             plan, as_stream(stream)))
    return rc;
  plan->first_pages = first_pages;
  plan->last_pages = last_pages;
  return PG_OK;
}

extern "C" int32_t pg_sparse_select(const pg_segment_plan_t* plan, const void* query, int64_t query_batch_stride,
                                    const void* bounds, const void* key_scale, const int32_t* indices,
                                    int32_t* selected, void* workspace, void* stream) {
  clear_error();
  if (!plan || !query || !selected || !workspace) return fail(PG_ERROR_INVALID_ARGUMENT, "null select argument");
  if (plan->selected_pages <= 0 || plan->batch_size <= 0 || plan->batch_size > 65535 || plan->num_kv_heads <= 0 ||
      plan->num_qo_heads % plan->num_kv_heads || plan->num_qo_heads / plan->num_kv_heads > 16)
    return fail(PG_ERROR_INVALID_ARGUMENT, "the plan is not one of pg_sparse_plan");
  if (plan->has_history && (!bounds || !key_scale || !indices))
    return fail(PG_ERROR_INVALID_ARGUMENT, "bounds, scales or tables missing");
  if (reinterpret_cast<uintptr_t>(query) % 16 || reinterpret_cast<uintptr_t>(bounds) % 16 || query_batch_stride % 8)
    return fail(PG_ERROR_INVALID_ARGUMENT, "queries and bounds must be 16-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  SelectArgs a{};
  a.query = static_cast<const uint16_t*>(query);
  a.query_batch_stride = query_batch_stride;
  a.bounds = static_cast<const uint8_t*>(bounds);
  a.key_scale = static_cast<const uint16_t*>(key_scale);
  a.indices = indices;
  a.indptr = reinterpret_cast<const int32_t*>(ws + plan->indptr_offset);
  a.scores = reinterpret_cast<float*>(ws + plan->scores_offset);
  a.selected = selected;
  a.take = plan->selected_pages;
  a.first = plan->first_pages;
  a.last = plan->last_pages;
  a.num_kv_heads = plan->num_kv_heads;
  a.group = plan->num_qo_heads / plan->num_kv_heads;
  hipStream_t s = as_stream(stream);
  if (plan->max_pages > plan->selected_pages) {
    const int64_t groups = (plan->max_pages + kScorePages - 1) / kScorePages;
    const int64_t waves = groups * plan->num_kv_heads * plan->batch_size;
    // more pages per wave, which has its query to prepare first, once there are waves
    // enough to keep every CU reading (45 uneven requests, 43000 pages of 4 heads: 12.5 us so,
    // 14.2 with twice the groups and 15.4 with half; 8 requests of 8192 pages, 134 MB of
    // bounds: 25.7, 25.6 and 28.4)
    a.wave_groups = static_cast<int>(std::min<int64_t>(kMostGroups, std::max<int64_t>(1, waves / 8192)));
    const int64_t block_groups = static_cast<int64_t>(a.wave_groups) * (kScoreThreads / kWave);
    hipLaunchKernelGGL(page_scores_kernel,
                       dim3(static_cast<unsigned>((groups + block_groups - 1) / block_groups), plan->num_kv_heads,
                            plan->batch_size),
                       dim3(kScoreThreads), 0, s, a);
    if (int32_t rc = check_launch("page_scores")) return rc;
  }
  const dim3 grid(plan->num_kv_heads, plan->batch_size), threads(kPickThreads);
  if (plan->max_pages <= 2 * kPickThreads)
    hipLaunchKernelGGL(pick_pages_kernel<2>, grid, threads, 0, s, a);
  else if (plan->max_pages <= 8 * kPickThreads)
    hipLaunchKernelGGL(pick_pages_kernel<8>, grid, threads, 0, s, a);
  else if (plan->max_pages <= 32 * kPickThreads)
    hipLaunchKernelGGL(pick_pages_kernel<32>, grid, threads, 0, s, a);
  else
    hipLaunchKernelGGL(pick_pages_kernel<0>, grid, threads, 0, s, a);
  return check_launch("pick_pages");
}

extern "C" int32_t pg_sparse_run(const pg_segment_plan_t* plan, const void* query, int64_t query_batch_stride,
                                 const void* key, const void* value, const void* key_scale,
                                 const void* value_scale, const int32_t* indices, const int32_t* last_page_len,
                                 const int32_t* selected, const void* tail_k, const void* tail_v,
                                 const int32_t* tail_indices, const int32_t* tail_last_len,
                                 const void* value_center, void* out, float* lse, float sm_scale,
                                 void* workspace, void* stream) {
  clear_error();
  if (!plan) return fail(PG_ERROR_INVALID_ARGUMENT, "null run argument");
  PageAttentionArgs a{};
  a.query = static_cast<const uint16_t*>(query);
  a.query_batch_stride = query_batch_stride;
  a.key = key;
  a.value = value;
  a.key_scale = static_cast<const uint16_t*>(key_scale);
  a.value_scale = static_cast<const uint16_t*>(value_scale);
  a.indices = indices;
  a.last_page_len = last_page_len;
  a.selected = selected;
  a.selected_pages = plan->selected_pages;
  a.tail_k = static_cast<const uint16_t*>(tail_k);
  a.tail_v = static_cast<const uint16_t*>(tail_v);
  a.tail_indices = tail_indices;
  a.tail_last = tail_last_len;
  a.value_center = static_cast<const uint16_t*>(value_center);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  if (int32_t rc = check_attention(*plan, a, sm_scale, workspace)) return rc;
  if (plan->selected_pages <= 0) return fail(PG_ERROR_INVALID_ARGUMENT, "the plan is not one of pg_sparse_plan");
  if (plan->has_history && !selected) return fail(PG_ERROR_INVALID_ARGUMENT, "no selection");
  place_work(*plan, workspace, sm_scale, a);
  const dim3 grid(static_cast<unsigned>(plan->num_items) * plan->num_kv_heads);
  hipStream_t s = as_stream(stream);
  if (a.group > kNarrowRows)
    hipLaunchKernelGGL(selected_attention_kernel<true>, grid, dim3(kAttentionThreads), 0, s, a);
  else
    hipLaunchKernelGGL(selected_attention_kernel<false>, grid, dim3(kAttentionThreads), 0, s, a);
  if (int32_t rc = check_launch("selected_attention")) return rc;
  return launch_combine(*plan, a, workspace, s);
}
