// Attention of single tokens over pages held in 4 bits and exact FP16 pages
// (layout: pg_int4.h), split over the context, with the value center added back.
//
//   out = sum_t p_t sV_t v_t / sum_t p_t + cV,  p_t = exp2(sm log2(e) sK_t q . k_t - m)
//
// over codes k, v in [-7, 7] and one scale per token, head and part.  The key
// center shifts all of a request's scores alike and is left out.
//
// A workgroup takes one KV head with its query heads and a range of pages; its 4
// waves take groups of 4 pages in turn and meet in LDS once, at the end.
// Everything else stays in registers, with hardly an exchange between lanes:
//  * QK as K Q^T: tokens are the MFMA's rows, heads its columns, so lane (kg, n)
//    gets the scores of tokens 4 kg .. 4 kg + 3 for head n % 8, or n where the KV
//    head has more than 8 (kWide).
//  * These are, pair of pages by pair, exactly the k slots that the lane feeds
//    as the A operand of P V: probabilities never leave their lane.  Columns
//    n < 8 hand over the FP16 part of a probability and columns n >= 8 (the same
//    heads again) its remainder, so rows r and r + 8 of the product add up to
//    one of about 23 bits.  With kWide the two parts are a product each (16 heads
//    per KV head, 256 requests: 188 us, as two workgroups of 8 heads 268).
//  * Codes are exact FP16 operands, normal ones: a nibble u = code + 8 is masked out
//    under an exponent and 1024 + 8 or 64 + 8 taken off, 2.5 operations per pair.  Masked
//    nibbles as they are, FP16 subnormals, would save one of these and cost the result:
//    the sums of an MFMA are cut at a width that counts from an operand's nominal
//    exponent, and subnormal ones lose the bits that they lack (6 to 7 % of the outputs
//    a step from the nearest FP16 value and lse 4e-6 to 5e-6 off, now 0.04 % at most and
//    6e-7); with V's offset of 8 also left to the product it was 15 to 18 %.  The
//    scales multiply scores and probabilities in float32.
//  * The softmax's base follows the running maximum lazily: it moves when a
//    score passes it by 2^4, so most groups of pages need no exchange at all.
//
// Probabilities times V's scales are carried relative to a power of two that
// puts the largest of the wave's scales near 2^10 (2^14 with the base's slack), so
// that two FP16 parts hold them to 2^-23 of themselves or 2^-35 of the largest.
//
// Bound by HBM once a wave has several groups, by a chain of trips to memory
// (work item, page ids, pages, partial rows) before.  Kernel times on MI355X, and
// of the same walk without its arithmetic: 256 requests (829 MB) 170 and 165 us,
// 8 requests of 4K to 32K (164 MB) 34 and 32, one of 49K tokens (53 MB) 14.9 and
// 12.4, of 4K (5 MB) 5.5 and 4.7; a join adds 2.4 to 4.6 us.  Measured and not
// taken: 8 waves a workgroup (one fits a CU, and nothing covers its start and
// end: 256 requests 191 us), and a join by the workgroup that ends last (49K
// tokens 18.7 us a call against 17.2 with the second launch, before the last
// steps: counting across XCDs costs what the launch does), and pages requested two
// groups ahead (19.0 us a call at 49K tokens against 16.6, 190 at 256 requests:
// the clamped or checked addresses cost more than the wait).
#include "pg_int4.h"
#include "pg_int4_plan.h"

#include <algorithm>

namespace pg {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint16_t v2s __attribute__((ext_vector_type(2)));

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kThreads = kWave * kInt4Waves;
constexpr int kNarrowHeads = 8;    // query heads whose probabilities' parts share a product

struct Int4Args {
  const uint16_t* query;
  int64_t query_batch_stride;
  const uint8_t* codes;
  const uint16_t* scales;
  const int32_t* indices;
  const int32_t* last_page_len;
  const uint16_t* tail_k;
  const uint16_t* tail_v;
  const int32_t* tail_indices;
  const int32_t* tail_last_len;
  const uint16_t* value_center;
  int64_t center_batch_stride;
  const Int4Item* items;
  float* partial_o;                // [items][Hq][128]
  float* partial_m;                // [items][Hq], base-2 scores
  float* partial_l;
  uint16_t* out;
  float* lse;
  float sm_scale_log2;
  int num_qo_heads, num_kv_heads, group;
};

__device__ __forceinline__ v2h as_half2(uint32_t bits) { return __builtin_bit_cast(v2h, bits); }

__device__ __forceinline__ v2s as_short2(uint32_t bits) { return __builtin_bit_cast(v2s, bits); }

__device__ __forceinline__ v8h operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(v8h, v4u{a, b, c, d});
}

// Codes of a dword in FP16, as 8 MFMA operands in their order: a nibble u = code + 8
// put under the exponent of 1024 (nibbles 0 and 4), or one nibble further up of 64 (1
// and 5), is 1024 + u or 64 + u, and less 1032 or 72 it is the code, exactly.  The
// exponents are held in registers: masking and putting is one operation that takes
// but one constant of another kind.
struct Exponents {
  uint32_t even = 0x64006400u, odd = 0x54005400u;
  __device__ __forceinline__ Exponents() { asm("" : "+v"(even), "+v"(odd)); }
  __device__ __forceinline__ uint32_t even_codes(uint32_t word) const {
    return __builtin_bit_cast(uint32_t, as_half2((word & 0x000f000fu) | even) - as_half2(0x64086408u));
  }
  __device__ __forceinline__ uint32_t odd_codes(uint32_t word) const {
    return __builtin_bit_cast(uint32_t, as_half2((word & 0x00f000f0u) | odd) - as_half2(0x54805480u));
  }
};

__device__ __forceinline__ v2h to_half2(float x, float y) {
  return __builtin_convertvector((v2f{x, y}), v2h);
}

// x times one half of ``pair``: one mixed-precision operation, no conversion.
__device__ __forceinline__ float times_half(float x, uint32_t pair, int which) {
  return fmaf(x, static_cast<float>(as_half2(pair)[which]), 0.0f);
}

constexpr float kSlack = 4.0f;     // how far (base 2) a score may pass the base

// Running state of one wave.  Lane (kg, n) has head n % 8's (kWide: n's): base (before the
// softmax scale), limit past which it moves, and offset, the exponent of the sums
// minus the scaled base; l sums the lane's own tokens.  acc[nb][r] is row 4 kg + r of
// the product, channel 8 n + nb.
struct State {
  float base, limit, offset;
  float l[2];                      // of tokens 4 kg, 4 kg + 1 and of the other two
  v4f acc[8];
};

__device__ __forceinline__ void scale_sums(State& st, const float (&f)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) st.acc[nb][r] *= f[r];
}

// Softmax step over kPages pages: s are the lane's scores, masked ones -inf,
// v_scale pairs of V's scales (FP16; 0 where masked), ``scale`` the softmax scale
// in base 2, ``exponent`` that of the sums.  p: the lane's rows of the A operand
// of P V, with kCodes times V's scales; rows of the FP16 part and of the remainder in
// one, or with kWide in one after the other.
template <int kPages, bool kCodes, bool kWide>
__device__ __forceinline__ void softmax_step(State& st, const float (&s)[kPages][4],
                                             const uint32_t (&v_scale)[kPages][2], float scale,
                                             float exponent, float low_part, int lane,
                                             v8h (&p)[1 + kWide][kPages / 2]) {
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kPages; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
  if (__builtin_amdgcn_ballot_w64(top > st.limit)) {
    top = fmaxf(top, __shfl_xor(top, 16, kWave));
    top = fmaxf(top, __shfl_xor(top, 32, kWave));
    const float base = fmaxf(st.base, top);
    // a head with nothing visible yet keeps a base of -inf and an offset of 0
    const float alpha = base == kNegInf ? 1.0f : __builtin_amdgcn_exp2f((st.base - base) * scale);
    st.base = base;
    st.limit = base + kSlack / scale;
    st.offset = base == kNegInf ? exponent : fmaf(-base, scale, exponent);
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
      const float x0 = __builtin_amdgcn_exp2f(fmaf(s[page][r], scale, st.offset));
      const float x1 = __builtin_amdgcn_exp2f(fmaf(s[page][r + 1], scale, st.offset));
      st.l[h & 1] += x0 + x1;
      const float w0 = kCodes ? times_half(x0, v_scale[page][h & 1], 0) : x0;
      const float w1 = kCodes ? times_half(x1, v_scale[page][h & 1], 1) : x1;
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

// The low or the high halves of two words, side by side.
__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t b, bool high) {
  return high ? __builtin_amdgcn_perm(b, a, 0x07060302u) : __builtin_amdgcn_perm(b, a, 0x05040100u);
}

// Pins ``x`` here: the wait for its load is placed at this point, not earlier.
template <typename T>
__device__ __forceinline__ void consume_point(T& x) {
  T value = x;
  asm volatile("" : "+v"(value));
  x = value;
}

struct Group {
  v4u k[kInt4GroupPages], v[kInt4GroupPages], s[kInt4GroupPages];
};

template <bool kWide>
__global__ __launch_bounds__(kThreads, 2) void int4_decode_kernel(Int4Args a) {
  constexpr int kHeads = kWide ? 16 : kNarrowHeads;
  __shared__ float part_o[kInt4Waves][kHeads][kHeadDim];
  __shared__ float part_m[kInt4Waves][kHeads];
  __shared__ float part_l[kInt4Waves][kHeads];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int n = lane & 15, kg = lane >> 4;
  const Int4Item it = a.items[blockIdx.x];
  const int kv = blockIdx.y, heads = a.group;
  const int hkv = a.num_kv_heads;

  // query: B operand, column n = head n % kHeads, dims 32 w + 8 kg ..; columns past
  // the heads repeat the first one and are dropped at the end
  v8h q[4];
  {
    const uint16_t* row = a.query + it.request * a.query_batch_stride +
                          static_cast<int64_t>(kv * a.group + (n % kHeads < heads ? n % kHeads : 0)) * kHeadDim;
#pragma unroll
    for (int w = 0; w < 4; ++w) q[w] = *reinterpret_cast<const v8h*>(row + 32 * w + 8 * kg);
  }
  auto take_query = [&]() {        // once the first pages are on their way
#pragma unroll
    for (int w = 0; w < 4; ++w) consume_point(q[w]);
  };
  const float low_part = kWide || n >= kHeads ? 1.0f : 0.0f;

  State st;
  st.base = st.limit = kNegInf;
  st.offset = st.l[0] = st.l[1] = 0.0f;
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) st.acc[nb] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  float exponent = 0.0f;           // of the sums l and acc

  // ---- history: groups wave, wave + 4, ... of the item's pages
  const int count = it.page_end - it.page_begin;
  const int all_groups = (count + kInt4GroupPages - 1) / kInt4GroupPages;
  const int groups = (all_groups - wave + kInt4Waves - 1) / kInt4Waves;
  if (groups > 0) {
    // lane l: slot l of the wave, page 4 (4 (l / 4) + wave) + l % 4 of the item
    const int slot_page = kInt4GroupPages * (kInt4Waves * (lane / kInt4GroupPages) + wave) +
                          lane % kInt4GroupPages;
    const int my_page = a.indices[it.page_begin + min(slot_page, count - 1)];
    const int last_len = min(a.last_page_len[it.request], kPageSize);
    auto visible = [&](int page) {     // tokens of the item's page ``page``
      return page >= count ? 0 : it.page_begin + page == it.last_page ? last_len : kPageSize;
    };
    const int whole = visible(count - 1) == kPageSize ? count : count - 1;   // leading whole pages
    // byte offset of the slot's block of codes; its scales are at 1/32 of that
    static_assert(kInt4BlockBytes == 32 * 2 * kInt4BlockScales, "scales of a block");
    const int64_t my_block = (static_cast<int64_t>(my_page) * hkv + kv) * kInt4BlockBytes;
    const int my_low = static_cast<int>(my_block), my_high = static_cast<int>(my_block >> 32);
    const uint32_t lane_bytes = 16 * lane, lane_scales = 16 * kg;
    const uint8_t* scale_bytes = reinterpret_cast<const uint8_t*>(a.scales);
    Group buf[2];
    auto issue = [&](int g, Group& dst) {
#pragma unroll
      for (int i = 0; i < kInt4GroupPages; ++i) {
        const int slot = g * kInt4GroupPages + i;
        const uint64_t block = static_cast<uint32_t>(__builtin_amdgcn_readlane(my_low, slot)) |
                               static_cast<uint64_t>(__builtin_amdgcn_readlane(my_high, slot)) << 32;
        const uint8_t* codes = a.codes + block;
        dst.k[i] = *reinterpret_cast<const v4u*>(codes + lane_bytes);
        dst.v[i] = *reinterpret_cast<const v4u*>(codes + kInt4PartBytes + lane_bytes);
        dst.s[i] = *reinterpret_cast<const v4u*>(scale_bytes + (block >> 5) + lane_scales);
      }
    };
    issue(0, buf[0]);
    // the largest visible V scale of the wave's pages fixes the power of two
    v2u raw[4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
      raw[g] = *reinterpret_cast<const v2u*>(scale_bytes + (my_block >> 5) + 16 * g + 8);
    take_query();
    {
      // positive FP16 values order as their bits do
      if (whole < count) {
        const int limit = visible(slot_page);
#pragma unroll
        for (int t = 0; t < kPageSize; t += 2)
          raw[t >> 2][(t & 3) >> 1] &= t + 1 < limit ? ~0u : t < limit ? 0x0000ffffu : 0u;
      }
      v2s top = as_short2(raw[0][0]);
#pragma unroll
      for (int d = 1; d < 8; ++d) top = __builtin_elementwise_max(top, as_short2(raw[d >> 1][d & 1]));
      float largest = fmaxf(half_bits_to_float(top.x), half_bits_to_float(top.y));
      largest = row16_max(largest);
      largest = fmaxf(largest, __shfl_xor(largest, 16, kWave));
      largest = fmaxf(largest, __shfl_xor(largest, 32, kWave));
      int e = 0;
      if (largest > 0.0f) frexpf(largest, &e);
      exponent = st.offset = static_cast<float>(10 - e);
    }

    const Exponents at;
    auto compute = [&](int g, Group& cur) {
      const int first = kInt4GroupPages * (kInt4Waves * g + wave);
      float s[kInt4GroupPages][4];
#pragma unroll
      for (int i = 0; i < kInt4GroupPages; ++i) {
        consume_point(cur.k[i]);
        consume_point(cur.s[i]);
        v4f dot = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t x = cur.k[i][w];
          dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              operand(at.even_codes(x), at.odd_codes(x), at.even_codes(x >> 8), at.odd_codes(x >> 8)), q[w], dot, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = times_half(dot[r], cur.s[i][r >> 1], r & 1);
      }
      uint32_t v_scale[kInt4GroupPages][2];
#pragma unroll
      for (int i = 0; i < kInt4GroupPages; ++i) {
        v_scale[i][0] = cur.s[i][2];
        v_scale[i][1] = cur.s[i][3];
      }
      if (first + kInt4GroupPages > whole) {     // a partial or a missing page
#pragma unroll
        for (int i = 0; i < kInt4GroupPages; ++i) {
          int limit = visible(first + i) - 4 * kg;
          consume_point(limit);     // keeps this a branch: whole groups skip the selects
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[i][r] = r < limit ? s[i][r] : kNegInf;
            v_scale[i][r >> 1] &= r < limit ? ~0u : r & 1 ? 0x0000ffffu : 0xffff0000u;
          }
        }
      }
      v8h p[1 + kWide][kInt4GroupPages / 2];
      softmax_step<kInt4GroupPages, true, kWide>(st, s, v_scale, a.sm_scale_log2, exponent, low_part, lane, p);
#pragma unroll
      for (int i = 0; i < kInt4GroupPages; ++i) consume_point(cur.v[i]);
      auto product = [&](const v8h (&rows)[1 + kWide], v8h columns, v4f sum) {
#pragma unroll
        for (int part = 0; part < 1 + kWide; ++part)
          sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(rows[part], columns, sum, 0, 0, 0);
        return sum;
      };
#pragma unroll
      for (int j = 0; j < kInt4GroupPages / 2; ++j) {
        v8h rows[1 + kWide];
#pragma unroll
        for (int part = 0; part < 1 + kWide; ++part) rows[part] = p[part][j];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t x = cur.v[2 * j][w], y = cur.v[2 * j + 1][w];
          st.acc[2 * w] = product(
              rows, operand(at.even_codes(x), at.odd_codes(x), at.even_codes(y), at.odd_codes(y)), st.acc[2 * w]);
          st.acc[2 * w + 1] = product(
              rows, operand(at.even_codes(x >> 8), at.odd_codes(x >> 8), at.even_codes(y >> 8), at.odd_codes(y >> 8)),
              st.acc[2 * w + 1]);
        }
      }
    };
    // the loads of group g + 1 are in flight while group g is computed
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
  } else {
    take_query();
  }

  // ---- exact tail: pairs wave, wave + 4, ... of the item's tail pages
  const int tail_count = it.tail_end - it.tail_begin;
  if (2 * wave < tail_count) {
    // probabilities alone: their largest is 1, or 2^4 with the base's slack
    const float change = __builtin_amdgcn_exp2f(10.0f - exponent);
    st.l[0] *= change;
    st.l[1] *= change;
    st.offset += 10.0f - exponent;
    const float f[4] = {change, change, change, change};
    scale_sums(st, f);
    exponent = 10.0f;
    const int64_t row_stride = static_cast<int64_t>(hkv) * kHeadDim;
    const int last_len = min(a.tail_last_len[it.request], kPageSize);
    for (int page = 2 * wave; page < tail_count; page += 2 * kInt4Waves) {
      float s[2][4];
      v4u k[2][4], v[2][4];
      int limit[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = it.tail_begin + min(page + i, tail_count - 1);
        const int64_t base = static_cast<int64_t>(a.tail_indices[at]) * kPageSize * row_stride + kv * kHeadDim;
        limit[i] = (page + i >= tail_count ? 0 : at == it.last_tail ? last_len : kPageSize) - 4 * kg;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          k[i][w] = *reinterpret_cast<const v4u*>(a.tail_k + base + n * row_stride + 32 * w + 8 * kg);
#pragma unroll
        for (int t = 0; t < 4; ++t)
          v[i][t] = *reinterpret_cast<const v4u*>(a.tail_v + base + (4 * kg + t) * row_stride + 8 * n);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v4f dot = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w)
          dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, k[i][w]), q[w], dot, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[i][r] = r < limit[i] ? dot[r] : kNegInf;
          // a row not yet written may hold anything: 0 times it must be 0
          if (r >= limit[i]) v[i][r] = v4u{0u, 0u, 0u, 0u};
        }
      }
      v8h p[1 + kWide][1];
      const uint32_t unscaled[2][2] = {};
      softmax_step<2, false, kWide>(st, s, unscaled, a.sm_scale_log2, exponent, low_part, lane, p);
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
        v4u cols;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          cols[2 * i] = pick(v[i][0][nb >> 1], v[i][1][nb >> 1], nb & 1);
          cols[2 * i + 1] = pick(v[i][2][nb >> 1], v[i][3][nb >> 1], nb & 1);
        }
#pragma unroll
        for (int part = 0; part < 1 + kWide; ++part)
          st.acc[nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[part][0], __builtin_bit_cast(v8h, cols), st.acc[nb], 0, 0, 0);
      }
    }
  }

  // ---- the waves meet: parts of the product's rows, then 4 partial states
  float l_sum = st.l[0] + st.l[1];
  l_sum += __shfl_xor(l_sum, 16, kWave);
  l_sum += __shfl_xor(l_sum, 32, kWave);
  const float scale = __builtin_amdgcn_exp2f(-exponent);
  if (kg == 0 && n < kHeads) {
    part_m[wave][n] = st.base * a.sm_scale_log2;
    part_l[wave][n] = l_sum * scale;
  }
  // part_o[..][64 b + c]: dim 2 c + b.  A swap of two registers' halves adds rows r
  // and r + 8 of two channels at once: lanes below 32 end with channel 8 n + 2 p, the
  // others with the next; with kWide rows are whole.
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (kWide) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        *reinterpret_cast<float4*>(&part_o[wave][(4 * kg + r) % kHeads][64 * b + 4 * n]) =
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
  // wave w finishes heads w, w + 4, two dims per lane
  for (int h = wave; h < heads; h += kInt4Waves) {
    float m = kNegInf;
#pragma unroll
    for (int w = 0; w < kInt4Waves; ++w) m = fmaxf(m, part_m[w][h]);
    const float base = m == kNegInf ? 0.0f : m;
    float l = 0.0f;
    float2 o = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kInt4Waves; ++w) {
      const float f = __builtin_amdgcn_exp2f(part_m[w][h] - base);
      const float2 x = make_float2(part_o[w][h][lane], part_o[w][h][64 + lane]);
      l += f * part_l[w][h];
      o.x += f * x.x;
      o.y += f * x.y;
    }
    const int head = kv * a.group + h;
    if (it.items_in_request > 1) {
      const int64_t row = static_cast<int64_t>(blockIdx.x) * a.num_qo_heads + head;
      *reinterpret_cast<float2*>(a.partial_o + row * kHeadDim + 2 * lane) = o;
      if (lane == 0) {
        a.partial_m[row] = m;
        a.partial_l[row] = l;
      }
      continue;
    }
    const int64_t row = static_cast<int64_t>(it.request) * a.num_qo_heads + head;
    float2 c = make_float2(0.0f, 0.0f);
    if (a.value_center) {
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(
          a.value_center + it.request * a.center_batch_stride + kv * kHeadDim + 2 * lane);
      c = make_float2(half_bits_to_float(static_cast<uint16_t>(bits)),
                      half_bits_to_float(static_cast<uint16_t>(bits >> 16)));
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;      // no token: the center alone
    *reinterpret_cast<__half2*>(a.out + row * kHeadDim + 2 * lane) =
        __floats2half2_rn(o.x * inv + c.x, o.y * inv + c.y);
    if (lane == 0 && a.lse) a.lse[row] = l == 0.0f ? kNegInf : log2f(l) + m;
  }
}

struct Int4CombineArgs {
  const float* partial_o;
  const float* partial_m;
  const float* partial_l;
  const int32_t* item_ptr;
  const uint16_t* value_center;
  int64_t center_batch_stride;
  uint16_t* out;
  float* lse;
  int num_qo_heads, group;
  int single;                      // one request: its items (item_ptr is not read)
};

// Joins the partial states of one (request, query head), 64 dims a workgroup:
// thread (row, column) = (tid / 16, tid % 16) takes items row, row + 16, ... of
// four dims.  The first 64 items are requested together, so a join of that many
// is one trip to memory after the item range.
constexpr int kCombineThreads = 256;
constexpr int kCombineRows = kCombineThreads / 16;
constexpr int kCombineInFlight = 4;

__global__ __launch_bounds__(kCombineThreads) void int4_combine_kernel(Int4CombineArgs a) {
  constexpr int kWaves = kCombineThreads / kWave;
  __shared__ float part_o[kWaves][64];
  __shared__ float part_m[kWaves], part_l[kWaves];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int row = threadIdx.x / 16, dim = 64 * blockIdx.z + 4 * (threadIdx.x % 16);
  const int request = blockIdx.x, head = blockIdx.y;
  const int begin = a.single ? 0 : a.item_ptr[request];
  const int end = a.single ? a.single : a.item_ptr[request + 1];
  if (end - begin <= 1) return;    // its only workgroup wrote the output
  float m = kNegInf, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int first = begin + row; first < end; first += kCombineRows * kCombineInFlight) {
    float mi[kCombineInFlight], li[kCombineInFlight];
    float4 x[kCombineInFlight];
#pragma unroll
    for (int k = 0; k < kCombineInFlight; ++k) {
      const int item = first + k * kCombineRows;
      const int64_t at = static_cast<int64_t>(min(item, end - 1)) * a.num_qo_heads + head;
      mi[k] = a.partial_m[at];
      li[k] = a.partial_l[at];
      x[k] = *reinterpret_cast<const float4*>(a.partial_o + at * kHeadDim + dim);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kCombineInFlight; ++k) {
      if (first + k * kCombineRows >= end) mi[k] = kNegInf;
      top = fmaxf(top, mi[k]);
    }
    const float base = top == kNegInf ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - base);
    l *= f;
    o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
    for (int k = 0; k < kCombineInFlight; ++k) {
      if (first + k * kCombineRows >= end) break;
      const float g = __builtin_amdgcn_exp2f(mi[k] - base);
      l = fmaf(g, li[k], l);
      o.x = fmaf(g, x[k].x, o.x);
      o.y = fmaf(g, x[k].y, o.y);
      o.z = fmaf(g, x[k].z, o.z);
      o.w = fmaf(g, x[k].w, o.w);
    }
    m = top;
  }
  // the wave's four rows, then the waves
  float top = fmaxf(m, __shfl_xor(m, 16, kWave));
  top = fmaxf(top, __shfl_xor(top, 32, kWave));
  const float base = top == kNegInf ? 0.0f : top;
  const float f = __builtin_amdgcn_exp2f(m - base);
  float sums[5] = {l * f, o.x * f, o.y * f, o.z * f, o.w * f};
#pragma unroll
  for (float& x : sums) {
    x += __shfl_xor(x, 16, kWave);
    x += __shfl_xor(x, 32, kWave);
  }
  if (lane < 16)
    *reinterpret_cast<float4*>(&part_o[wave][4 * lane]) = make_float4(sums[1], sums[2], sums[3], sums[4]);
  if (lane == 0) {
    part_m[wave] = top;
    part_l[wave] = sums[0];
  }
  __syncthreads();
  if (wave != 0) return;
  float all = kNegInf;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all = fmaxf(all, part_m[w]);
  const float all_base = all == kNegInf ? 0.0f : all;
  float sum = 0.0f, out = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float g = __builtin_amdgcn_exp2f(part_m[w] - all_base);
    sum = fmaf(g, part_l[w], sum);
    out = fmaf(g, part_o[w][lane], out);
  }
  const int64_t at = static_cast<int64_t>(request) * a.num_qo_heads + head;
  const int d = 64 * blockIdx.z + lane;
  const float center = a.value_center ? half_bits_to_float(a.value_center[
      request * a.center_batch_stride + (head / a.group) * kHeadDim + d]) : 0.0f;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  a.out[at * kHeadDim + d] = __half_as_ushort(__float2half_rn(out * inv + center));
  if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? kNegInf : log2f(sum) + all;
}

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_int4_plan(const int32_t* host_indptr, const int32_t* host_tail_indptr,
                                int32_t batch_size, int32_t num_qo_heads, int32_t num_kv_heads,
                                int32_t num_cus, void* workspace, int64_t workspace_bytes,
                                pg_int4_plan_t* plan, void* stream) {
  clear_error();
  if (!plan || !workspace) return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  return guarded([&]() -> int32_t {
    std::vector<Int4Item> items;
    std::vector<int32_t> item_ptr;
    pg_int4_plan_t p{};
    if (int32_t rc = build_int4_plan(host_indptr, host_tail_indptr, batch_size, num_qo_heads,
                                     num_kv_heads, num_cus, items, item_ptr, p))
      return rc;
    if (p.workspace_bytes > workspace_bytes)
      return fail(PG_ERROR_WORKSPACE, "decode workspace too small: need " +
                                          std::to_string(p.workspace_bytes) + " bytes, have " +
                                          std::to_string(workspace_bytes));
    hipStream_t s = as_stream(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (hipMemcpyAsync(ws + p.items_offset, items.data(), items.size() * sizeof(Int4Item),
                       hipMemcpyHostToDevice, s) != hipSuccess ||
        hipMemcpyAsync(ws + p.item_ptr_offset, item_ptr.data(), item_ptr.size() * sizeof(int32_t),
                       hipMemcpyHostToDevice, s) != hipSuccess ||
        hipStreamSynchronize(s) != hipSuccess)
      return fail(PG_ERROR_LAUNCH, "plan copy failed");
    *plan = p;
    return PG_OK;
  });
}

extern "C" int32_t pg_int4_decode_run(const pg_int4_plan_t* plan, const void* query,
                                      int64_t query_batch_stride, const void* codes,
                                      const void* scales, const int32_t* indices,
                                      const int32_t* last_page_len, const void* tail_k,
                                      const void* tail_v, const int32_t* tail_indices,
                                      const int32_t* tail_last_len, const void* value_center,
                                      int64_t center_batch_stride, void* out, float* lse,
                                      float sm_scale, void* workspace, void* stream) {
  clear_error();
  if (!plan || !query || !out || !workspace) return fail(PG_ERROR_INVALID_ARGUMENT, "null run argument");
  if (plan->has_history && (!codes || !scales || !indices || !last_page_len))
    return fail(PG_ERROR_INVALID_ARGUMENT, "history segment tensors missing");
  if (plan->has_tail && (!tail_k || !tail_v || !tail_indices || !tail_last_len))
    return fail(PG_ERROR_INVALID_ARGUMENT, "tail segment tensors missing");
  // the kernel multiplies it by log2(e), and scores of any FP16 values by that
  if (!(sm_scale > 0.0f) || !(sm_scale < 0x1p100f))
    return fail(PG_ERROR_INVALID_ARGUMENT, "sm_scale must be positive and below 2^100");
  for (const void* p : {query, codes, scales, tail_k, tail_v})
    if (reinterpret_cast<uintptr_t>(p) % 16)
      return fail(PG_ERROR_INVALID_ARGUMENT, "queries and pages must be 16-byte aligned");
  if (query_batch_stride % 8) return fail(PG_ERROR_INVALID_ARGUMENT, "query rows must be 16-byte aligned");
  for (const void* p : {value_center, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(p) % 4)
      return fail(PG_ERROR_INVALID_ARGUMENT, "centers and outputs must be 4-byte aligned");
  if (plan->num_items <= 0 || plan->batch_size <= 0 || plan->num_kv_heads <= 0 ||
      plan->num_qo_heads % plan->num_kv_heads || plan->num_qo_heads / plan->num_kv_heads > 16)
    return fail(PG_ERROR_INVALID_ARGUMENT, "the plan is not one of pg_int4_plan");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Int4Args a{};
  a.query = static_cast<const uint16_t*>(query);
  a.query_batch_stride = query_batch_stride;
  a.codes = static_cast<const uint8_t*>(codes);
  a.scales = static_cast<const uint16_t*>(scales);
  a.indices = indices;
  a.last_page_len = last_page_len;
  a.tail_k = static_cast<const uint16_t*>(tail_k);
  a.tail_v = static_cast<const uint16_t*>(tail_v);
  a.tail_indices = tail_indices;
  a.tail_last_len = tail_last_len;
  a.value_center = static_cast<const uint16_t*>(value_center);
  a.center_batch_stride = center_batch_stride;
  a.items = reinterpret_cast<const Int4Item*>(ws + plan->items_offset);
  const int64_t rows = static_cast<int64_t>(plan->num_items) * plan->num_qo_heads;
  a.partial_o = reinterpret_cast<float*>(ws + plan->partial_offset);
  a.partial_m = a.partial_o + rows * kHeadDim;
  a.partial_l = a.partial_m + rows;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.sm_scale_log2 = sm_scale * 1.4426950408889634f;
  a.num_qo_heads = plan->num_qo_heads;
  a.num_kv_heads = plan->num_kv_heads;
  a.group = plan->num_qo_heads / plan->num_kv_heads;
  const dim3 grid(plan->num_items, plan->num_kv_heads);
  if (a.group <= kNarrowHeads)
    hipLaunchKernelGGL(int4_decode_kernel<false>, grid, dim3(kThreads), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(int4_decode_kernel<true>, grid, dim3(kThreads), 0, as_stream(stream), a);
  if (int32_t rc = check_launch("int4_decode")) return rc;
  if (plan->max_items_per_request <= 1) return PG_OK;
  Int4CombineArgs c{};
  c.partial_o = a.partial_o;
  c.partial_m = a.partial_m;
  c.partial_l = a.partial_l;
  c.item_ptr = reinterpret_cast<const int32_t*>(ws + plan->item_ptr_offset);
  c.value_center = a.value_center;
  c.center_batch_stride = center_batch_stride;
  c.out = a.out;
  c.lse = lse;
  c.num_qo_heads = plan->num_qo_heads;
  c.group = a.group;
  c.single = plan->batch_size == 1 ? plan->num_items : 0;
  hipLaunchKernelGGL(int4_combine_kernel, dim3(plan->batch_size, plan->num_qo_heads, kHeadDim / 64),
                     dim3(kCombineThreads), 0, as_stream(stream), c);
  return check_launch("int4_combine");
}
