// Attention of up to 16 query rows over a list of pages, INT8 or FP16, and exact FP16
// pages: the part that attention over shared prefixes (pg_prefix.hip) and over selected
// pages (pg_sparse.hip) have in common.
//
//   out = sum_t p_t v_t / sum_t p_t + cV,   p_t = exp2(sm log2(e) q . k_t - m)
//
// An INT8 key or value is code * scale, one scale per page and KV head.  The key center
// shifts all of a request's scores alike and is left out; the value center is added at
// the end.
//
// A workgroup takes one KV head and a work item; its 4 waves take groups of 4 pages (INT8)
// or pairs (FP16) in turn and meet in LDS once, at the end.  Within a wave nothing leaves
// the registers:
//  * QK as K Q^T: tokens are the rows of v_mfma_f32_16x16x32_f16, query rows its columns,
//    so lane (kg, n) gets the scores of tokens 4 kg .. 4 kg + 3 for query row n % 8, or n
//    where there are more than 8 (kWide).
//  * These are, pair of pages by pair, the k slots that the lane feeds as the A operand of
//    P V.  Probabilities go in as an FP16 part and its remainder, about 23 bits together:
//    in columns n < 8 and n >= 8 of one product, or with kWide in a product each.
//  * INT8 codes are exact FP16 operands: a byte c put as c ^ 0x80 under the exponent of 1024
//    is 1024 + 128 + c, and less 1152 it is c.  Two values take a permutation of bytes, half
//    an exclusive or (a whole one for V, whose token pairs come from two rows) and a packed
//    subtraction.  Scales multiply scores and probabilities in float32.
//  * The softmax's base follows the running maximum lazily: it moves when a score passes it
//    by 2^4, so most groups of pages need no exchange between lanes.
//
// Bound by HBM once a wave has several groups, by a chain of trips to memory (work item, page
// ids, pages, partial rows) before: 512 workgroups over 256 picked pages of 8 requests' 8 heads
// and their 128 exact pages, 75 MB, 19 to 21 us (3.5 to 4.0 TB/s: a head's rows are lines of 128 bytes apart
// from each other); 256 requests of 6 to 63 INT8 and 16 exact pages, 558 MB, about 125 us (4.5 TB/s);
// 2000 tokens of 4 requests 8.3 us.  Measured and not taken: partial rows' slots requested
// ahead of the pages (the first of these 19.3 us: registers).
#pragma once

#include "pg_combine.h"
#include "pg_segment_plan.h"

#include <algorithm>
#include <cstring>

namespace pg {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kAttentionThreads = kWave * kSegmentWaves;
constexpr float kSlack = 4.0f;       // how far (base 2) a score may pass the base
constexpr float kExactExponent = 10.0f;   // of the sums over exact pages

struct PageAttentionArgs {
  const uint16_t* query;
  int64_t query_batch_stride;
  const void* key;                   // pages [*, 16, Hkv, 128], INT8 or FP16
  const void* value;
  const uint16_t* key_scale;         // [*, Hkv], INT8 only
  const uint16_t* value_scale;
  const int32_t* prefix_indices;
  const int32_t* prefix_last;        // per segment
  const int32_t* indices;
  const int32_t* last_page_len;      // per request
  const int32_t* selected;           // [B, Hkv, selected_pages] positions in a request's table
  int32_t selected_pages;
  const uint16_t* tail_k;
  const uint16_t* tail_v;
  const int32_t* tail_indices;
  const int32_t* tail_last;
  const uint16_t* value_center;      // [B, Hkv, 128]
  const SegmentItem* items;
  const int32_t* slot_base;
  float* partial_o;                  // [slots][Hq][128]
  float* partial_m;                  // [slots][Hq], base-2 scores
  float* partial_l;
  uint16_t* out;
  float* lse;
  float sm_scale_log2;
  float slack;                       // how far a score, not yet scaled, may pass the base
  int num_qo_heads, num_kv_heads, group;
};

__device__ __forceinline__ v2h as_half2(uint32_t bits) { return __builtin_bit_cast(v2h, bits); }

__device__ __forceinline__ v8h operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(v8h, v4u{a, b, c, d});
}

__device__ __forceinline__ uint32_t minus_1152(uint32_t pair) {
  return __builtin_bit_cast(uint32_t, as_half2(pair) - as_half2(0x64806480u));
}

// Bytes 0, 1 or 2, 3 of ``word`` (codes ^ 0x80) in FP16.
__device__ __forceinline__ uint32_t low_codes(uint32_t word) {
  return minus_1152(__builtin_amdgcn_perm(0x64646464u, word, 0x04010400u));
}
__device__ __forceinline__ uint32_t high_codes(uint32_t word) {
  return minus_1152(__builtin_amdgcn_perm(0x64646464u, word, 0x04030402u));
}

// Byte ``at`` of two rows side by side in FP16.
__device__ __forceinline__ uint32_t column_codes(uint32_t row0, uint32_t row1, int at) {
  return minus_1152(__builtin_amdgcn_perm(row1, row0, 0x0c040c00u + 0x00010001u * at) ^ 0x64806480u);
}

// The low or the high halves of two words, side by side.
__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t b, bool high) {
  return high ? __builtin_amdgcn_perm(b, a, 0x07060302u) : __builtin_amdgcn_perm(b, a, 0x05040100u);
}

__device__ __forceinline__ v2h to_half2(float x, float y) {
  return __builtin_convertvector((v2f{x, y}), v2h);
}

// Running state of one wave.  Lane (kg, n) has query row n % 8's (kWide: n's): base (before
// the softmax scale), and shift, which is the base or 0 before there is one; l sums the
// lane's own tokens.  acc[nb][r] is row 4 kg + r of the product, channel 8 n + nb.
struct RowState {
  float base, shift;
  float l[2];
  v4f acc[8];
};

__device__ __forceinline__ void scale_sums(RowState& st, const float (&f)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) st.acc[nb][r] *= f[r];
}

// Softmax step over kPages pages: s are the lane's scores, masked ones -inf, v_scale the
// pages' V scales (with kScaled), ``scale`` the softmax scale in base 2, ``exponent`` that
// of the sums.  The base comes off the scores before they are scaled: past 2^24 a product less
// the rounded product of the base could be anything (fused the other way an operation less per
// score: 61 requests over FP16 pages 33.5 us, 34.1 so; over INT8 pages the same).
// p: the lane's rows of the A operand of P V; the FP16 part and the remainder in one, or with
// kWide in one after the other.
template <int kPages, bool kScaled, bool kWide>
__device__ __forceinline__ void softmax_step(RowState& st, const float (&s)[kPages][4],
                                             const float (&v_scale)[kPages], float scale, float slack,
                                             float exponent, float low_part, int lane, v8h (&p)[1 + kWide][kPages / 2]) {
  float top = kNoScore;
#pragma unroll
  for (int i = 0; i < kPages; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
  if (__builtin_amdgcn_ballot_w64(top - st.base > slack)) {
    top = fmaxf(top, __shfl_xor(top, 16, kWave));
    top = fmaxf(top, __shfl_xor(top, 32, kWave));
    const float base = fmaxf(st.base, top);
    // a row with nothing visible yet keeps a base of -inf
    const float alpha = base == kNoScore ? 1.0f : __builtin_amdgcn_exp2f((st.base - base) * scale);
    st.base = base;
    st.shift = base == kNoScore ? 0.0f : base;
    st.l[0] *= alpha;
    st.l[1] *= alpha;
    const int kg = lane >> 4;
    float f[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = __shfl(alpha, (4 * kg + r) & (kWide ? 15 : 7), kWave);
    scale_sums(st, f);
  }
#pragma unroll
  for (int j = 0; j < kPages / 2; ++j) {
    uint32_t words[1 + kWide][4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int page = 2 * j + (h >> 1), r = 2 * (h & 1);
      const float x0 = __builtin_amdgcn_exp2f(fmaf(s[page][r] - st.shift, scale, exponent));
      const float x1 = __builtin_amdgcn_exp2f(fmaf(s[page][r + 1] - st.shift, scale, exponent));
      st.l[h & 1] += x0 + x1;
      const float w0 = kScaled ? x0 * v_scale[page] : x0;
      const float w1 = kScaled ? x1 * v_scale[page] : x1;
      // the FP16 part, or what it leaves, each to nearest: together within 2^-23
      const v2h high = to_half2(w0, w1);
      if (kWide) words[0][h] = __builtin_bit_cast(uint32_t, high);
      words[kWide][h] = __builtin_bit_cast(uint32_t, to_half2(
          fmaf(-low_part, static_cast<float>(high.x), w0), fmaf(-low_part, static_cast<float>(high.y), w1)));
    }
#pragma unroll
    for (int part = 0; part < 1 + kWide; ++part)
      p[part][j] = operand(words[part][0], words[part][1], words[part][2], words[part][3]);
  }
}

// Pins ``x`` here: the wait for its load is placed at this point, not earlier.
template <typename T>
__device__ __forceinline__ void consume_point(T& x) {
  T value = x;
  asm volatile("" : "+v"(value));
  x = value;
}

template <bool kWide>
__device__ __forceinline__ v4f product(const v8h (&rows)[1 + kWide], v8h columns, v4f sum) {
#pragma unroll
  for (int part = 0; part < 1 + kWide; ++part)
    sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(rows[part], columns, sum, 0, 0, 0);
  return sum;
}

// What a lane knows of the page in its slot: slot 4 g + i of a wave is page i of its g-th
// group, 4 (4 g + wave) + i of the item (kGroup = 4; pairs with kGroup = 2).
template <int kGroup>
__device__ __forceinline__ int slot_page(int lane, int wave) {
  return kGroup * (kSegmentWaves * (lane / kGroup) + wave) + lane % kGroup;
}

__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(x), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(
             __builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane))) << 32 | low);
}

// Runs step(g, buffer) for g = 0 .. groups - 1, the loads of group g + 1 in flight.
template <typename Buffer, typename Issue, typename Compute>
__device__ __forceinline__ void pipelined(int groups, Buffer (&buf)[2], Issue&& issue, Compute&& compute) {
  int g = 0;
  for (; g + 2 < groups; g += 2) {
    issue(g + 1, buf[1]);
    compute(g, buf[0]);
    issue(g + 2, buf[0]);
    compute(g + 1, buf[1]);
  }
  if (g + 1 < groups) {
    issue(g + 1, buf[1]);
    compute(g, buf[0]);
    compute(g + 1, buf[1]);
  } else {
    compute(g, buf[0]);
  }
}

struct CodeGroup {
  v4u k[kSegmentGroupPages][2];
  v2u v[kSegmentGroupPages][4];
};

struct ExactPair {
  v4u k[2][4], v[2][4];
};

// Pages of FP16 K and V: the wave's pairs of ``count`` pages, lane's slot at page ``my_page``
// with ``my_visible`` tokens.
template <bool kWide>
__device__ __forceinline__ void exact_pages(RowState& st, const v8h (&q)[4], const uint16_t* key,
                                            const uint16_t* value, int count, int my_page, int my_visible,
                                            int kv, int hkv, float scale, float slack, float low_part, int wave,
                                            int lane) {
  const int n = lane & 15, kg = lane >> 4;
  const int all = (count + 1) / 2;
  const int groups = (all - wave + kSegmentWaves - 1) / kSegmentWaves;
  const uint32_t row_bytes = static_cast<uint32_t>(hkv) * kHeadDim * 2;
  const uint32_t k_lane = n * row_bytes + kv * kHeadDim * 2 + 16 * kg;
  const uint32_t v_lane = 4 * kg * row_bytes + kv * kHeadDim * 2 + 16 * n;
  const int64_t my_base = static_cast<int64_t>(my_page) * kPageSize * row_bytes;
  const uint8_t* k_bytes = reinterpret_cast<const uint8_t*>(key);
  const uint8_t* v_bytes = reinterpret_cast<const uint8_t*>(value);
  ExactPair buf[2];
  auto issue = [&](int g, ExactPair& dst) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t base = lane_value(my_base, 2 * g + i);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        dst.k[i][w] = *reinterpret_cast<const v4u*>(k_bytes + base + k_lane + 64 * w);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        dst.v[i][t] = *reinterpret_cast<const v4u*>(v_bytes + base + v_lane + t * row_bytes);
    }
  };
  auto compute = [&](int g, ExactPair& cur) {
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int limit = __builtin_amdgcn_readlane(my_visible, 2 * g + i) - 4 * kg;
      v4f dot = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
        dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, cur.k[i][w]), q[w], dot, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = r < limit ? dot[r] : kNoScore;
        // a row not yet written may hold anything: 0 times it must be 0
        if (r >= limit) cur.v[i][r] = v4u{0u, 0u, 0u, 0u};
      }
    }
    v8h p[1 + kWide][1];
    const float unscaled[2] = {};
    softmax_step<2, false, kWide>(st, s, unscaled, scale, slack, kExactExponent, low_part, lane, p);
    v8h rows[1 + kWide];
#pragma unroll
    for (int part = 0; part < 1 + kWide; ++part) rows[part] = p[part][0];
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[2 * i] = pick(cur.v[i][0][nb >> 1], cur.v[i][1][nb >> 1], nb & 1);
        w[2 * i + 1] = pick(cur.v[i][2][nb >> 1], cur.v[i][3][nb >> 1], nb & 1);
      }
      st.acc[nb] = product<kWide>(rows, operand(w[0], w[1], w[2], w[3]), st.acc[nb]);
    }
  };
  issue(0, buf[0]);
  pipelined(groups, buf, issue, compute);
}

// What the waves of a workgroup meet in.
template <bool kWide>
struct NarrowMeeting {
  static constexpr int kRows = kWide ? 16 : kNarrowRows;
  float o[kSegmentWaves][kRows][kHeadDim];
  float m[kSegmentWaves][kRows];
  float l[kSegmentWaves][kRows];
};

template <bool kCodes, bool kSelected, bool kWide>
__device__ __forceinline__ void page_attention(const PageAttentionArgs& a, const SegmentItem& it, int kv,
                                               NarrowMeeting<kWide>& meet) {
  constexpr int kRows = NarrowMeeting<kWide>::kRows;
  auto& part_o = meet.o;
  auto& part_m = meet.m;
  auto& part_l = meet.l;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int n = lane & 15, kg = lane >> 4;
  const int hkv = a.num_kv_heads;

  // query rows: B operand, column n = row n % kRows, dims in the order of K's loads;
  // columns past the rows repeat the first one and are dropped at the end
  auto dims = [&](int w) { return kCodes ? 32 * kg + 8 * w : 32 * w + 8 * kg; };
  v8h q[4];
  const uint16_t* q_row;
  {
    const int row = it.row_first + (n % kRows < it.rows ? n % kRows : 0);
    q_row = a.query + (it.request + row / a.group) * a.query_batch_stride +
            static_cast<int64_t>(kv * a.group + row % a.group) * kHeadDim;
#pragma unroll
    for (int w = 0; w < 4; ++w) q[w] = *reinterpret_cast<const v8h*>(q_row + dims(w));
  }
  const float low_part = kWide || n >= kRows ? 1.0f : 0.0f;

  RowState st;
  st.base = kNoScore;
  st.shift = st.l[0] = st.l[1] = 0.0f;
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) st.acc[nb] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  float exponent = 0.0f;             // of the sums l and acc

  // ---- history: the wave's groups of the item's pages
  constexpr int kGroup = kCodes ? kSegmentGroupPages : 2;
  const int count = it.page_end - it.page_begin;
  if (kGroup * wave < count) {
    const int at = slot_page<kGroup>(lane, wave);
    const int listed = it.page_begin + min(at, count - 1);
    const int last_len = min(it.segment >= 0 ? a.prefix_last[it.segment] : a.last_page_len[it.request], kPageSize);
    int my_page, my_visible;
    if (kSelected) {
      const int position = a.selected[(static_cast<int64_t>(it.request) * hkv + kv) * a.selected_pages + listed];
      const bool valid = position >= 0 && position < it.table_pages;
      my_page = a.indices[it.table_begin + (valid ? position : 0)];
      my_visible = !valid ? 0 : position == it.table_pages - 1 ? last_len : kPageSize;
    } else {
      my_page = (it.segment >= 0 ? a.prefix_indices : a.indices)[listed];
      my_visible = listed == it.last_page ? last_len : kPageSize;
    }
    // an entry below 0 is no page: the pool's first one is read in its place, and weighs nothing
    if (at >= count || my_page < 0) my_visible = 0;
    my_page = max(my_page, 0);
    if constexpr (!kCodes) {
      exponent = kExactExponent;
      exact_pages<kWide>(st, q, static_cast<const uint16_t*>(a.key), static_cast<const uint16_t*>(a.value), count,
                         my_page, my_visible, kv, hkv, a.sm_scale_log2, a.slack, low_part, wave, lane);
    } else {
      const int all_groups = (count + kGroup - 1) / kGroup;
      const int groups = (all_groups - wave + kSegmentWaves - 1) / kSegmentWaves;
      const uint32_t row_bytes = static_cast<uint32_t>(hkv) * kHeadDim;
      const uint32_t k_lane = n * row_bytes + kv * kHeadDim + 32 * kg;
      const uint32_t v_lane = 4 * kg * row_bytes + kv * kHeadDim + 8 * n;
      const int64_t my_base = static_cast<int64_t>(my_page) * kPageSize * row_bytes;
      const uint8_t* k_bytes = static_cast<const uint8_t*>(a.key);
      const uint8_t* v_bytes = static_cast<const uint8_t*>(a.value);
      CodeGroup buf[2];
      auto issue = [&](int g, CodeGroup& dst) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const int64_t base = lane_value(my_base, kGroup * g + i);
#pragma unroll
          for (int w = 0; w < 2; ++w)
            dst.k[i][w] = *reinterpret_cast<const v4u*>(k_bytes + base + k_lane + 16 * w);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            dst.v[i][t] = *reinterpret_cast<const v2u*>(v_bytes + base + v_lane + t * row_bytes);
        }
      };
      issue(0, buf[0]);
      const int64_t my_scale = static_cast<int64_t>(my_page) * hkv + kv;
      const float my_k_scale = half_bits_to_float(a.key_scale[my_scale]);
      // a page that is not visible weighs nothing, whatever its scale
      const float my_v_scale = my_visible > 0 ? half_bits_to_float(a.value_scale[my_scale]) : 0.0f;
      // Probabilities times V's scales are carried relative to a power of two that puts
      // the largest of the wave's scales near 2^10 (2^14 with the base's slack), so that two
      // FP16 parts hold them to 2^-23 of themselves or 2^-35 of the largest.
      {
        float largest = row16_max(fabsf(my_v_scale));
        largest = fmaxf(largest, __shfl_xor(largest, 16, kWave));
        largest = fmaxf(largest, __shfl_xor(largest, 32, kWave));
        int e = 0;
        if (largest > 0.0f && largest < -kNoScore) frexpf(largest, &e);
        exponent = static_cast<float>(10 - e);
      }
      auto compute = [&](int g, CodeGroup& cur) {
        float s[kGroup][4], v_scale[kGroup];
        int least = kPageSize;
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const int slot = kGroup * g + i;
          consume_point(cur.k[i][0]);
          consume_point(cur.k[i][1]);
          const float k_scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_k_scale), slot));
          v_scale[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_v_scale), slot));
          least = min(least, __builtin_amdgcn_readlane(my_visible, slot));
          v4f dot = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x = cur.k[i][w >> 1][2 * (w & 1)] ^ 0x80808080u;
            const uint32_t y = cur.k[i][w >> 1][2 * (w & 1) + 1] ^ 0x80808080u;
            dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                operand(low_codes(x), high_codes(x), low_codes(y), high_codes(y)), q[w], dot, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][r] = dot[r] * k_scale;
        }
        if (least < kPageSize) {       // a partial or a missing page
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            int limit = __builtin_amdgcn_readlane(my_visible, kGroup * g + i) - 4 * kg;
            consume_point(limit);      // keeps this a branch: whole groups skip the selects
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] = r < limit ? s[i][r] : kNoScore;
          }
        }
        v8h p[1 + kWide][kGroup / 2];
        softmax_step<kGroup, true, kWide>(st, s, v_scale, a.sm_scale_log2, a.slack, exponent, low_part, lane, p);
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) consume_point(cur.v[i][t]);
#pragma unroll
        for (int j = 0; j < kGroup / 2; ++j) {
          v8h rows[1 + kWide];
#pragma unroll
          for (int part = 0; part < 1 + kWide; ++part) rows[part] = p[part][j];
#pragma unroll
          for (int nb = 0; nb < 8; ++nb) {
            const int word = nb >> 2, byte = nb & 3;
            const v2u (&x)[4] = cur.v[2 * j];
            const v2u (&y)[4] = cur.v[2 * j + 1];
            st.acc[nb] = product<kWide>(
                rows, operand(column_codes(x[0][word], x[1][word], byte), column_codes(x[2][word], x[3][word], byte),
                              column_codes(y[0][word], y[1][word], byte), column_codes(y[2][word], y[3][word], byte)),
                st.acc[nb]);
          }
        }
      };
      pipelined(groups, buf, issue, compute);
    }
  }

  // ---- exact tail: the wave's pairs of the item's tail pages
  const int tail_count = it.tail_end - it.tail_begin;
  if (2 * wave < tail_count) {
    // probabilities alone: their largest is 1, or 2^4 with the base's slack
    const float change = __builtin_amdgcn_exp2f(kExactExponent - exponent);
    st.l[0] *= change;
    st.l[1] *= change;
    const float f[4] = {change, change, change, change};
    scale_sums(st, f);
    exponent = kExactExponent;
    if (kCodes) {
#pragma unroll
      for (int w = 0; w < 4; ++w) q[w] = *reinterpret_cast<const v8h*>(q_row + 32 * w + 8 * kg);
    }
    const int at = slot_page<2>(lane, wave);
    const int listed = it.tail_begin + min(at, tail_count - 1);
    const int my_page = a.tail_indices[listed];
    int my_visible = listed == it.last_tail ? min(a.tail_last[it.request], kPageSize) : kPageSize;
    if (at >= tail_count || my_page < 0) my_visible = 0;
    exact_pages<kWide>(st, q, a.tail_k, a.tail_v, tail_count, max(my_page, 0), my_visible, kv, hkv, a.sm_scale_log2,
                       a.slack, low_part, wave, lane);
  }

  // ---- the waves meet: parts of the product's rows, then 4 partial states
  float l_sum = st.l[0] + st.l[1];
  l_sum += __shfl_xor(l_sum, 16, kWave);
  l_sum += __shfl_xor(l_sum, 32, kWave);
  const float scale = __builtin_amdgcn_exp2f(-exponent);
  if (kg == 0 && n < kRows) {
    part_m[wave][n] = st.base * a.sm_scale_log2;
    part_l[wave][n] = l_sum * scale;
  }
  // part_o[..][64 b + c]: dim 2 c + b.  A swap of two registers' halves adds rows r and
  // r + 8 of two channels at once: lanes below 32 end with channel 8 n + 2 p, the others
  // with the next; with kWide rows are whole.
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (kWide) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        *reinterpret_cast<float4*>(&part_o[wave][(4 * kg + r) % kRows][64 * b + 4 * n]) =
            make_float4(st.acc[b][r] * scale, st.acc[2 + b][r] * scale, st.acc[4 + b][r] * scale,
                        st.acc[6 + b][r] * scale);
      continue;
    }
    float o[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const v2u x = __builtin_amdgcn_permlane32_swap(__float_as_uint(st.acc[2 * p][r]),
                                                     __float_as_uint(st.acc[2 * p + 1][r]), false, false);
      o[p] = (__uint_as_float(x.x) + __uint_as_float(x.y)) * scale;
    }
    *reinterpret_cast<float4*>(&part_o[wave][4 * (kg & 1) + r][64 * (lane >> 5) + 4 * n]) =
        make_float4(o[0], o[1], o[2], o[3]);
  }
  __syncthreads();
  // wave w finishes rows w, w + 4, ..., two dims per lane
  for (int h = wave; h < it.rows; h += kSegmentWaves) {
    float m = kNoScore;
#pragma unroll
    for (int w = 0; w < kSegmentWaves; ++w) m = fmaxf(m, part_m[w][h]);
    const float base = m == kNoScore ? 0.0f : m;
    float l = 0.0f;
    float2 o = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kSegmentWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(part_m[w][h] - base);
      const float2 x = make_float2(part_o[w][h][lane], part_o[w][h][64 + lane]);
      l += f * part_l[w][h];
      o.x += f * x.x;
      o.y += f * x.y;
    }
    const int in_segment = (it.row_first + h) / a.group;
    const int request = it.request + in_segment;
    const int head = kv * a.group + (it.row_first + h) % a.group;
    if (it.slot_at >= 0) {
      const int64_t slot = a.slot_base[it.slot_at + in_segment] + it.split;
      const int64_t row = slot * a.num_qo_heads + head;
      *reinterpret_cast<float2*>(a.partial_o + row * kHeadDim + 2 * lane) = o;
      if (lane == 0) {
        a.partial_m[row] = m;
        a.partial_l[row] = l;
      }
      continue;
    }
    const int64_t row = static_cast<int64_t>(request) * a.num_qo_heads + head;
    float2 c = make_float2(0.0f, 0.0f);
    if (a.value_center) {
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(
          a.value_center + (static_cast<int64_t>(request) * hkv + kv) * kHeadDim + 2 * lane);
      c = make_float2(half_bits_to_float(static_cast<uint16_t>(bits)),
                      half_bits_to_float(static_cast<uint16_t>(bits >> 16)));
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;       // no token: the center alone
    *reinterpret_cast<__half2*>(a.out + row * kHeadDim + 2 * lane) =
        __floats2half2_rn(o.x * inv + c.x, o.y * inv + c.y);
    if (lane == 0 && a.lse) a.lse[row] = l == 0.0f ? kNoScore : log2f(l) + m;
  }
}

// What both entry points take alike; ``kind``'s and the plan's own are theirs to check.
inline int32_t check_attention(const pg_segment_plan_t& plan, const PageAttentionArgs& a, float sm_scale,
                               const void* workspace) {
  if (!a.query || !a.out || !workspace) return fail(PG_ERROR_INVALID_ARGUMENT, "null run argument");
  const bool pages = plan.has_history || plan.has_prefix;
  if (pages && (!a.key || !a.value || (plan.kind == PG_KV_INT8 && (!a.key_scale || !a.value_scale))))
    return fail(PG_ERROR_INVALID_ARGUMENT, "history pages missing");
  if (plan.has_history && (!a.indices || !a.last_page_len))
    return fail(PG_ERROR_INVALID_ARGUMENT, "history tables missing");
  if (plan.has_prefix && (!a.prefix_indices || !a.prefix_last))
    return fail(PG_ERROR_INVALID_ARGUMENT, "prefix tables missing");
  if (plan.has_tail && (!a.tail_k || !a.tail_v || !a.tail_indices || !a.tail_last))
    return fail(PG_ERROR_INVALID_ARGUMENT, "tail segment tensors missing");
  // times log2(e) and a score, which comes to 2^46 with codes and scales, it stays in float32
  if (!(sm_scale > 0.0f) || !(sm_scale < 0x1p80f))
    return fail(PG_ERROR_INVALID_ARGUMENT, "sm_scale must be positive and below 2^80");
  for (const void* p : {static_cast<const void*>(a.query), a.key, a.value, static_cast<const void*>(a.tail_k),
                        static_cast<const void*>(a.tail_v)})
    if (reinterpret_cast<uintptr_t>(p) % 16)
      return fail(PG_ERROR_INVALID_ARGUMENT, "queries and pages must be 16-byte aligned");
  if (a.query_batch_stride % 8) return fail(PG_ERROR_INVALID_ARGUMENT, "query rows must be 16-byte aligned");
  for (const void* p : {static_cast<const void*>(a.value_center), static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(p) % 4)
      return fail(PG_ERROR_INVALID_ARGUMENT, "centers and outputs must be 4-byte aligned");
  if (plan.num_items <= 0 || plan.batch_size <= 0 || plan.num_kv_heads <= 0 ||
      plan.num_qo_heads % plan.num_kv_heads || plan.num_qo_heads / plan.num_kv_heads > 16)
    return fail(PG_ERROR_INVALID_ARGUMENT, "the plan is not one of this entry point");
  return PG_OK;
}

inline void place_work(const pg_segment_plan_t& plan, void* workspace, float sm_scale, PageAttentionArgs& a) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.items = reinterpret_cast<const SegmentItem*>(ws + plan.items_offset);
  a.slot_base = reinterpret_cast<const int32_t*>(ws + plan.slot_base_offset);
  const int64_t rows = plan.partial_rows * plan.num_qo_heads;
  a.partial_o = reinterpret_cast<float*>(ws + plan.partial_offset);
  a.partial_m = a.partial_o + rows * kHeadDim;
  a.partial_l = a.partial_m + rows;
  a.sm_scale_log2 = sm_scale * 1.4426950408889634f;
  a.slack = std::min(kSlack / a.sm_scale_log2, __FLT_MAX__);
  a.num_qo_heads = plan.num_qo_heads;
  a.num_kv_heads = plan.num_kv_heads;
  a.group = plan.num_qo_heads / plan.num_kv_heads;
}

// Joins few partial rows of many requests: a wave per (request, query head), two dims a lane,
// 8 rows requested at once.  Workgroups of combine_kernel, which take half a pair's dims and
// 64 rows at once, are too many and too empty then (8192 pairs of 5 rows: 14.4 us, 7.9 so; 1952
// pairs of up to 15: 6.6 and 4.9); of few pairs those are the shorter trip (32 pairs of 8 rows:
// 3.3 us, 4.3 with 4 rows at once here).  With more rows per pair neither is the faster (2048
// pairs of 18).
constexpr int kFewRows = 8;
constexpr int kFewSlots = 16;
constexpr int64_t kManyPairs = 1024;

__global__ __launch_bounds__(kCombineThreads) void combine_few_kernel(CombineArgs a, int64_t pairs) {
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * (kCombineThreads / kWave) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (pair >= pairs) return;
  const int lane = threadIdx.x % kWave;
  const int64_t request = pair / a.num_qo_heads;
  const int head = static_cast<int>(pair - request * a.num_qo_heads);
  const int begin = a.item_ptr[request], end = a.item_ptr[request + 1];
  if (begin == end) return;          // its only workgroup wrote the output
  float m = kNoScore, l = 0.0f;
  float2 o = make_float2(0.0f, 0.0f);
  for (int first = begin; first < end; first += kFewRows) {
    float mi[kFewRows], li[kFewRows];
    float2 x[kFewRows];
#pragma unroll
    for (int k = 0; k < kFewRows; ++k) {
      mi[k] = kNoScore;
      if (first + k >= end) continue;
      const int64_t at = static_cast<int64_t>(first + k) * a.num_qo_heads + head;
      mi[k] = a.partial_m[at];
      li[k] = a.partial_l[at];
      x[k] = *reinterpret_cast<const float2*>(a.partial_o + at * kHeadDim + 2 * lane);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kFewRows; ++k) top = fmaxf(top, mi[k]);
    const float base = top == kNoScore ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - base);
    l *= f;
    o = make_float2(o.x * f, o.y * f);
#pragma unroll
    for (int k = 0; k < kFewRows; ++k) {
      if (first + k >= end) break;
      const float g = __builtin_amdgcn_exp2f(mi[k] - base);
      l = fmaf(g, li[k], l);
      o.x = fmaf(g, x[k].x, o.x);
      o.y = fmaf(g, x[k].y, o.y);
    }
    m = top;
  }
  float2 c = make_float2(0.0f, 0.0f);
  if (a.value_center) {
    const uint32_t bits = *reinterpret_cast<const uint32_t*>(
        a.value_center + request * a.center_batch_stride + (head / a.group) * kHeadDim + 2 * lane);
    c = make_float2(half_bits_to_float(static_cast<uint16_t>(bits)), half_bits_to_float(static_cast<uint16_t>(bits >> 16)));
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<__half2*>(a.out + pair * kHeadDim + 2 * lane) = __floats2half2_rn(o.x * inv + c.x, o.y * inv + c.y);
  if (lane == 0 && a.lse) a.lse[pair] = l == 0.0f ? kNoScore : log2f(l) + m;
}

// Joins the requests that have partial rows; the others' workgroups wrote the output.
inline int32_t launch_combine(const pg_segment_plan_t& plan, const PageAttentionArgs& a, const void* workspace,
                              hipStream_t stream) {
  if (plan.max_slots == 0) return PG_OK;
  CombineArgs c{};
  c.partial_o = a.partial_o;
  c.partial_m = a.partial_m;
  c.partial_l = a.partial_l;
  c.item_ptr = reinterpret_cast<const int32_t*>(static_cast<const uint8_t*>(workspace) + plan.slot_ptr_offset);
  c.value_center = a.value_center;
  c.center_batch_stride = static_cast<int64_t>(a.num_kv_heads) * kHeadDim;
  c.out = a.out;
  c.lse = a.lse;
  c.num_qo_heads = a.num_qo_heads;
  c.group = a.group;
  c.single = plan.batch_size == 1 ? plan.max_slots : 0;
  c.written = 0;
  const int64_t pairs = static_cast<int64_t>(plan.batch_size) * plan.num_qo_heads;
  if (plan.max_slots <= kFewSlots && pairs >= kManyPairs) {
    constexpr int kPairs = kCombineThreads / kWave;
    if (pairs > static_cast<int64_t>(UINT32_MAX) / kWave - kPairs)
      return fail(PG_ERROR_UNSUPPORTED, "too many requests for one launch");
    hipLaunchKernelGGL(combine_few_kernel, dim3(static_cast<unsigned>((pairs + kPairs - 1) / kPairs)),
                       dim3(kCombineThreads), 0, stream, c, pairs);
  } else {
    hipLaunchKernelGGL(combine_kernel, dim3(plan.batch_size, plan.num_qo_heads, kHeadDim / 64),
                       dim3(kCombineThreads), 0, stream, c);
  }
  return check_launch("combine");
}

// Plans on the host and copies the work list into the workspace.
inline int32_t plan_into(const SegmentBatch& batch, void* workspace, int64_t workspace_bytes,
                         pg_segment_plan_t* plan, hipStream_t stream) {
  if (!plan || !workspace) return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  return guarded([&]() -> int32_t {
    SegmentWork work;
    pg_segment_plan_t p{};
    if (int32_t rc = build_segment_plan(batch, work, p)) return rc;
    if (p.workspace_bytes > workspace_bytes)
      return fail(PG_ERROR_WORKSPACE, "decode workspace too small: need " + std::to_string(p.workspace_bytes) +
                                          " bytes, have " + std::to_string(workspace_bytes));
    // the tables lie in front of the workspace, one after the other: one copy
    std::vector<uint8_t> tables(p.scores_offset);
    auto put = [&](int64_t offset, const void* from, size_t bytes) {
      if (bytes) std::memcpy(tables.data() + offset, from, bytes);
    };
    put(p.items_offset, work.items.data(), work.items.size() * sizeof(SegmentItem));
    put(p.slot_ptr_offset, work.slot_ptr.data(), work.slot_ptr.size() * sizeof(int32_t));
    put(p.slot_base_offset, work.slot_base.data(), work.slot_base.size() * sizeof(int32_t));
    put(p.indptr_offset, batch.indptr, batch.selected > 0 ? work.slot_ptr.size() * sizeof(int32_t) : 0);
    if (hipMemcpyAsync(workspace, tables.data(), tables.size(), hipMemcpyHostToDevice, stream) != hipSuccess ||
        hipStreamSynchronize(stream) != hipSuccess)
      return fail(PG_ERROR_LAUNCH, "plan copy failed");
    *plan = p;
    return PG_OK;
  });
}

}  // namespace
}  // namespace pg
