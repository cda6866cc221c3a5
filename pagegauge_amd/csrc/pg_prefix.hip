// Attention of single tokens over prefixes that requests share, their own pages and an
// exact tail: each prefix's pages are read once for all of its requests.
#include "pg_page_attention.h"

namespace pg {
namespace {

typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

#define PG_LDS __attribute__((address_space(3)))

constexpr int kTileTokens = 64;
constexpr int kTilePages = kTileTokens / kPageSize;
constexpr int kTileBytes = kTileTokens * kHeadDim * 2;   // 16 KiB of FP16
constexpr float kRescaleLimit = 8.0f;                    // log2
// Probabilities are 2^7 times what the running maximum makes them, so at most 2^15 where it
// lags: as far up in FP16's range as goes, for the small ones' sake.
constexpr float kProbabilityExponent = 7.0f;
// A maximum past which scores are scaled before it comes off them: the product that it was
// rounded from may be further above it than FP16's range allows, from 2^24 on.
// A row that has seen nothing, or an infinity, has no part in that: other rows keep their bits.
constexpr float kLargeScore = 0x1p20f;
constexpr float kNoSuchScore = 0x1p127f;
// The running maximum before the first score.  Finite, so that a tile of -inf scores adds
// probabilities of 0 and not exp2(-inf + inf).
constexpr float kLowest = -__FLT_MAX__;

// LDS of a workgroup over shared rows: K0 K1 V0 V1, and the item's pages.
struct SharedTiles {
  uint8_t tiles[4 * kTileBytes];
  int32_t ids[kSharedMaxPages];                          // below 0: no page, the pool's first one is read
  float k_scale[kSharedMaxPages];
  float v_scale[kSharedMaxPages];
  float largest[kSegmentWaves];
  int32_t plain[kSegmentWaves];                          // no K scale below 0, no id either
};

// A prefix's pages with more than 32 query rows: kRowWaves waves of 32 query rows share
// every tile of 64 tokens through LDS, as FP16.
//
// A wave keeps its query rows as the B operand of v_mfma_f32_32x32x16_f16 and computes
// S^T = K Q^T, so that a lane holds scores of ONE row: the softmax reduces in registers plus
// one swap with the lane 32 away, and the probabilities are, register for register, the B
// operand of O^T += V^T P^T (V^T through transposing LDS reads).  With 4 waves of rows each
// takes the whole tile; with 2 the other two waves take the other 32 tokens of it, into
// partial rows of their own.
//
// INT8 codes become FP16 once, on their way into LDS, for all rows; K's scales multiply
// scores and V's the probabilities, a page (16 tokens) being one step of the product over
// tokens.  Probabilities times V's scales go in as one FP16 value, each off by 2^-11 of itself at
// most, or by 2^-32 of what the largest scale could weigh (V's scales count from the power of
// two at the item's largest).  An output is so off by up to 2^-11 of sum p |v|: where values do
// not cancel that is its own rounding, with values around zero and no center outputs are 2.9e-4
// off instead of 2.1e-4 (two in five are not the nearest FP16 value), and where values cancel it
// is all that is left.  With the remainder as a second part, which the form of up to 32 rows
// has, 256 requests on 16384 tokens take 185 us instead of 171 a call, the prefix alone 127
// instead of 107 (over FP16 pages 129): that costs more than it gives.
//
// Tiles go from memory to registers a whole iteration before they are put in LDS.
//
// Bound by the matrix cores and the VALU together: of the cycles of 256 requests (1024 query
// rows per KV head) over 16384 tokens MFMA takes 32 %, the VALU 48 % (36 and 39 % over FP16
// pages), LDS 35 %, and the two waves of a SIMD hide little of one behind the other.  69 GFLOP,
// 8 parts: 95 us over INT8 pages (723 TFLOP/s; the median of 30 in a row 102), 86 over FP16
// ones (797; 98; a library product of 8192 cubed reaches 1194); 48 query rows per KV head 19 us.
// Measured and not taken, beside 91 us at the time: the scores of
// tile j + 1 beside the softmax of tile j (one wave's 256 registers just hold it: 102 us),
// orders of instructions for the scheduler (97 to 104), no wave priority (93.8), priority to
// one of a CU's workgroups (96), V's scales in the exponents (the same with an eighth fewer
// vector operations), another swizzle without V's conflicts on the way into LDS (the same),
// tiles of 16 rows throughout (341).
template <bool kCodes, int kRowWaves>
__device__ __forceinline__ void shared_attention(const PageAttentionArgs& a, const SegmentItem& it, int kv,
                                                 SharedTiles& lds) {
  constexpr int kBlocks = kRowWaves == 4 ? 2 : 1;        // of 32 tokens, per wave and tile
  constexpr int kSteps = 2 * kBlocks;                    // pages, per wave and tile
  constexpr int kLoads = kCodes ? 2 : 4;                 // of 16 bytes, per thread, tile and tensor
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int half = lane >> 5, column = lane & 31;
  const int hkv = a.num_kv_heads;
  const int part = wave / kRowWaves;
  const int row_wave = 32 * (wave % kRowWaves);
  const int count = it.page_end - it.page_begin;
  const int tiles = (count + kTilePages - 1) / kTilePages;

  // tokens of the item that are visible: all but those past the prefix's last one
  const int last_len = it.page_end - 1 == it.last_page ? max(min(a.prefix_last[it.segment], kPageSize), 0) : kPageSize;
  const int visible = (count - 1) * kPageSize + last_len;
  // the item's pages; missing ones of the last tile repeat its last page, masked below, and a
  // page without a visible token counts with scales of 0, whatever its own are
  {
    const int32_t* table = a.prefix_indices + it.page_begin;
    float largest = 0.0f;
    bool plain = true;
    for (int i = threadIdx.x; i < tiles * kTilePages; i += kAttentionThreads) {
      const int32_t id = table[min(i, count - 1)];
      lds.ids[i] = id;
      plain &= id >= 0;
      if (kCodes) {
        const int64_t at = static_cast<int64_t>(max(id, 0)) * hkv + kv;
        const bool seen = i * kPageSize < visible && id >= 0;
        const float v = seen ? half_bits_to_float(a.value_scale[at]) : 0.0f;
        const float k = seen ? half_bits_to_float(a.key_scale[at]) * a.sm_scale_log2 : 0.0f;
        plain &= k >= 0.0f;
        lds.k_scale[i] = k;
        lds.v_scale[i] = v;
        if (fabsf(v) < -kNoScore) largest = fmaxf(largest, fabsf(v));
      }
    }
    if (kCodes) {
      largest = wave_max(largest);
      if (lane == 0) lds.largest[wave] = largest;
    }
    const bool all = !__builtin_amdgcn_ballot_w64(!plain);
    if (lane == 0) lds.plain[wave] = all;
  }
  const int row = it.row_first + min(row_wave + column, it.rows - 1);
  const int in_segment = row / a.group, head = kv * a.group + row % a.group;
  v8h qf[8];
  {
    const uint16_t* qp = a.query + (it.request + in_segment) * a.query_batch_stride + head * kHeadDim + 8 * half;
#pragma unroll
    for (int k = 0; k < 8; ++k) qf[k] = *reinterpret_cast<const v8h*>(qp + 16 * k);
  }
  __syncthreads();
  float v_unit = 1.0f, v_back = 1.0f;                    // 2^-e and 2^e of V's scales
  const bool plain = __builtin_amdgcn_readfirstlane(lds.plain[0] & lds.plain[1] & lds.plain[2] & lds.plain[3]);
  if (kCodes) {
    float largest = lds.largest[0];
#pragma unroll
    for (int w = 1; w < kSegmentWaves; ++w) largest = fmaxf(largest, lds.largest[w]);
    int e = 0;
    if (largest > 0.0f) frexpf(largest, &e);
    v_unit = __builtin_amdgcn_exp2f(static_cast<float>(-e));
    v_back = __builtin_amdgcn_exp2f(static_cast<float>(e));
  }

  // ---- tiles: thread t brings 16 bytes of rows t / 8 and 32 on (FP16: t / 16 and 16, 32, 48
  // on), so a wave's rows are of one page each time; the 16-byte chunks of a row in LDS are
  // swizzled by the row so that neither the K reads (8 rows per access) nor the transposing
  // V reads (4 rows x 32 bytes) meet in a bank
  const uint32_t element = kCodes ? 1 : 2;
  const uint32_t row_bytes = static_cast<uint32_t>(hkv) * kHeadDim * element;
  const int64_t page_bytes = static_cast<int64_t>(kPageSize) * row_bytes;
  const int my_row = threadIdx.x / (kCodes ? 8 : 16), my_chunk = threadIdx.x % (kCodes ? 8 : 16);
  const uint32_t from = (my_row % kPageSize) * row_bytes + kv * kHeadDim * element + 16 * my_chunk;
  const uint8_t* k_bytes = static_cast<const uint8_t*>(a.key);
  const uint8_t* v_bytes = static_cast<const uint8_t*>(a.value);
  auto page_at = [&](int tile, int i) { return kTilePages * tile + (kCodes ? 2 * i + (wave >> 1) : i); };
  v4u kr[kLoads], vr[kLoads];
  auto load = [&](const uint8_t* bytes, int tile, v4u (&r)[kLoads]) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int id = __builtin_amdgcn_readfirstlane(max(lds.ids[page_at(tile, i)], 0));
      r[i] = *reinterpret_cast<const v4u*>(bytes + id * page_bytes + from);
    }
  };
  auto store = [&](uint8_t* tile, const v4u (&r)[kLoads], int swizzle_mask, int swizzle_times) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int to = my_row + (kCodes ? 32 : 16) * i;
      const int swizzle = (to & swizzle_mask) * swizzle_times;
      uint8_t* at = tile + to * 256;
      if (kCodes) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = r[i][2 * h] ^ 0x80808080u, y = r[i][2 * h + 1] ^ 0x80808080u;
          *reinterpret_cast<v4u*>(at + (((2 * my_chunk + h) ^ swizzle) << 4)) =
              v4u{low_codes(x), high_codes(x), low_codes(y), high_codes(y)};
        }
      } else {
        *reinterpret_cast<v4u*>(at + ((my_chunk ^ swizzle) << 4)) = r[i];
      }
    }
  };
  auto load_k = [&](int tile) { load(k_bytes, tile, kr); };
  auto load_v = [&](int tile) { load(v_bytes, tile, vr); };
  auto store_k = [&](int buffer) { store(lds.tiles + buffer * kTileBytes, kr, 15, 1); };
  auto store_v = [&](int tile, int buffer) {
    if (!kCodes && (tile == tiles - 1 || !plain)) {      // rows not written may hold anything
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        if (kTileTokens * tile + my_row + 16 * i >= visible || lds.ids[page_at(tile, i)] < 0)
          vr[i] = v4u{0u, 0u, 0u, 0u};
    }
    store(lds.tiles + (2 + buffer) * kTileBytes, vr, 3, 4);
  };

  // LDS read offsets
  const uint32_t k_at = part * 8192 + column * 256 + ((half ^ (column & 15)) << 4);
  uint32_t v_at[4];
  {
    const int i = lane & 15, g = lane >> 4;
    const int v_row = 4 * (g >> 1) + (i >> 2);
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int chunk = 4 * d + 2 * (g & 1) + ((i & 3) >> 1);
      v_at[d] = 2 * kTileBytes + part * 8192 + v_row * 256 + ((chunk ^ (4 * (v_row & 3))) << 4) + 8 * (i & 1);
    }
  }

  v16f o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  float m = kLowest, l0 = 0.0f, l1 = 0.0f;

  auto qk = [&](int buffer, v16f (&s)[kBlocks]) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const v8h kf = *reinterpret_cast<const v8h*>(lds.tiles + (k_at ^ 32 * k) + buffer * kTileBytes + b * 8192);
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[k], s[b], 0, 0, 0);
      }
  };
  // factors of the wave's pages of a tile: K's scale with the softmax's, V's in its unit
  auto factors = [&](int tile, float (&kf)[kSteps], float (&vf)[kSteps]) {
#pragma unroll
    for (int p = 0; p < kSteps; ++p) {
      kf[p] = kCodes ? lds.k_scale[kTilePages * tile + 2 * part + p] : a.sm_scale_log2;
      vf[p] = kCodes ? lds.v_scale[kTilePages * tile + 2 * part + p] * v_unit : 1.0f;
    }
  };
  // the largest of the scores, once per row
  auto maximum = [&](const v16f (&s)[kBlocks], const float (&kf)[kSteps]) {
    float mx = kNoScore;
#pragma unroll
    for (int p = 0; p < kSteps; ++p) {
      float top = s[p / 2][8 * (p % 2)];
#pragma unroll
      for (int r = 1; r < 8; ++r) top = fmaxf(top, s[p / 2][8 * (p % 2) + r]);
      mx = fmaxf(mx, top * kf[p]);
    }
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  };
  auto raise = [&](float mx) {
    if (__builtin_amdgcn_ballot_w64(mx > m + kRescaleLimit)) {
      const float m_new = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l0 *= alpha;
      l1 *= alpha;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
  };
  // probabilities page by page, each followed by its product
  auto attend = [&](int buffer, const v16f (&s)[kBlocks], const float (&kf)[kSteps], const float (&vf)[kSteps]) {
    const float offset = kProbabilityExponent - m;
#pragma unroll
    for (int p = 0; p < kSteps; ++p) {
      v8h pr;
#pragma unroll
      for (int r = 0; r < 8; r += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[p / 2][8 * (p % 2) + r], kf[p], offset));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[p / 2][8 * (p % 2) + r + 1], kf[p], offset));
        l0 += p0;
        l1 += p1;
        pr[r] = static_cast<_Float16>(kCodes ? p0 * vf[p] : p0);
        pr[r + 1] = static_cast<_Float16>(kCodes ? p1 * vf[p] : p1);
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint8_t* at = lds.tiles + v_at[d] + buffer * kTileBytes + p * 4096;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PG_LDS v4s*)at);
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PG_LDS v4s*)(at + 2048));
        const v8h columns = __builtin_shufflevector(__builtin_bit_cast(v4h, lo), __builtin_bit_cast(v4h, hi),
                                                    0, 1, 2, 3, 4, 5, 6, 7);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(columns, pr, o[d], 0, 0, 0);
      }
    }
  };
  // iteration j: tile j is in LDS, tile j + 1 on its way to registers
  v16f s[kBlocks];
  auto stage_next = [&](int j, int buffer) {
    store_k(buffer ^ 1);
    store_v(j + 1, buffer ^ 1);
    // past the end the last tile comes again, and is not used
    const int next = min(j + 2, tiles - 1);
    load_k(next);
    load_v(next);
  };
  // the products each by itself, not within the sum with the base
  auto scale_scores = [&](float (&kf)[kSteps]) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = s[b][r] * kf[2 * b + r / 8];
        consume_point(x);
        s[b][r] = x;
      }
#pragma unroll
    for (int p = 0; p < kSteps; ++p) kf[p] = 1.0f;
  };
  // tiles without a masked token or a missing page
  auto body = [&](int j, int buffer) {
    __syncthreads();
    float kf[kSteps], vf[kSteps];
    factors(j, kf, vf);
    __builtin_amdgcn_s_setprio(1);
    qk(buffer, s);
    __builtin_amdgcn_s_setprio(0);
    stage_next(j, buffer);
    const float mx = maximum(s, kf);
    raise(mx);
    if (__builtin_amdgcn_ballot_w64(fabsf(m) > kLargeScore && fabsf(m) < kNoSuchScore)) scale_scores(kf);
    __builtin_amdgcn_s_setprio(1);
    attend(buffer, s, kf, vf);
    __builtin_amdgcn_s_setprio(0);
  };
  auto masked_body = [&](int j, int buffer) {
    __syncthreads();
    if (j + 1 < tiles) stage_next(j, buffer);
    float kf[kSteps], vf[kSteps];
    factors(j, kf, vf);
    qk(buffer, s);
    scale_scores(kf);
    int end[kSteps];                                     // of what is visible, for the wave's pages
#pragma unroll
    for (int p = 0; p < kSteps; ++p) end[p] = lds.ids[kTilePages * j + 2 * part + p] < 0 ? 0 : visible;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int token = kTileTokens * j + 32 * (part + b) + 8 * (r / 4) + 4 * half + r % 4;
        s[b][r] = token < end[2 * b + r / 8] ? s[b][r] : kNoScore;
      }
    const float mx = maximum(s, kf);
    raise(mx);
    attend(buffer, s, kf, vf);
  };

  load_k(0);
  load_v(0);
  store_k(0);
  store_v(0, 0);
  if (tiles > 1) {
    load_k(1);
    load_v(1);
  }
  // the largest score of a page is that of its largest product, unless a scale is negative;
  // with a missing page every tile is looked at
  int j = 0;
  if (plain)
    for (; j + 1 < tiles; ++j) body(j, j & 1);
  for (; j < tiles; ++j) masked_body(j, j & 1);

  if (row_wave + column >= it.rows) return;
  float l = l0 + l1;
  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  const int64_t slot = a.slot_base[it.slot_at + in_segment] + it.split + part;
  const int64_t to = slot * a.num_qo_heads + head;
  if (half == 0) {
    a.partial_m[to] = l == 0.0f ? kNoScore : m - kProbabilityExponent;
    a.partial_l[to] = l;
  }
  float* out = a.partial_o + to * kHeadDim + 4 * half;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<float4*>(out + 32 * d + 2 * r) =
          make_float4(o[d][r] * v_back, o[d][r + 1] * v_back, o[d][r + 2] * v_back, o[d][r + 3] * v_back);
}

// The forms share a launch, so that the matrix cores' work on shared prefixes and the
// reading of requests' own pages run side by side: 256 requests on 16384 tokens with 100 to
// 1000 of their own and 256 exact ones, 587 MB and 72 GFLOP, 162 to 180 us, where the prefix takes 95
// alone and the rest about 125.
template <bool kCodes>
__global__ __launch_bounds__(kAttentionThreads, 2) void prefix_attention_kernel(PageAttentionArgs a) {
  __shared__ __attribute__((aligned(1024))) union {
    SharedTiles tiles;
    NarrowMeeting<true> wide;
    NarrowMeeting<false> narrow;
  } lds;
  // KV heads vary fastest: with 8 of them each XCD reads one head's lines
  const SegmentItem it = a.items[blockIdx.x / a.num_kv_heads];
  const int kv = blockIdx.x % a.num_kv_heads;
  // tests of one value, each with a return: joined in another way their registers do not fit
  if (it.block_rows == 4 * kSharedRows) {
    shared_attention<kCodes, 4>(a, it, kv, lds.tiles);
    return;
  }
  if (it.block_rows == 2 * kSharedRows) {
    shared_attention<kCodes, 2>(a, it, kv, lds.tiles);
    return;
  }
  if (it.block_rows == kSegmentRows) {
    page_attention<kCodes, false, true>(a, it, kv, lds.wide);
    return;
  }
  if (it.block_rows == kNarrowRows) {
    page_attention<kCodes, false, false>(a, it, kv, lds.narrow);
    return;
  }
}

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_prefix_plan(const int32_t* host_prefix_requests, const int32_t* host_prefix_indptr,
                                  int32_t segments, const int32_t* host_indptr, const int32_t* host_tail_indptr,
                                  int32_t batch_size, int32_t num_qo_heads, int32_t num_kv_heads, int32_t kind,
                                  int32_t num_cus, void* workspace, int64_t workspace_bytes,
                                  pg_segment_plan_t* plan, void* stream) {
  clear_error();
  return plan_into({host_prefix_requests, host_prefix_indptr, segments, host_indptr, host_tail_indptr, batch_size,
                    num_qo_heads, num_kv_heads, kind, 0, num_cus}, workspace, workspace_bytes, plan,
                   as_stream(stream));
}

extern "C" int32_t pg_prefix_run(const pg_segment_plan_t* plan, const void* query, int64_t query_batch_stride,
                                 const void* key, const void* value, const void* key_scale,
                                 const void* value_scale, const int32_t* prefix_indices,
                                 const int32_t* prefix_last_len, const int32_t* indices,
                                 const int32_t* last_page_len, const void* tail_k, const void* tail_v,
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
  a.prefix_indices = prefix_indices;
  a.prefix_last = prefix_last_len;
  a.indices = indices;
  a.last_page_len = last_page_len;
  a.tail_k = static_cast<const uint16_t*>(tail_k);
  a.tail_v = static_cast<const uint16_t*>(tail_v);
  a.tail_indices = tail_indices;
  a.tail_last = tail_last_len;
  a.value_center = static_cast<const uint16_t*>(value_center);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  if (int32_t rc = check_attention(*plan, a, sm_scale, workspace)) return rc;
  if (plan->selected_pages) return fail(PG_ERROR_INVALID_ARGUMENT, "the plan is not one of pg_prefix_plan");
  place_work(*plan, workspace, sm_scale, a);
  const dim3 grid(static_cast<unsigned>(plan->num_items) * plan->num_kv_heads);
  hipStream_t s = as_stream(stream);
  if (plan->kind == PG_KV_INT8)
    hipLaunchKernelGGL(prefix_attention_kernel<true>, grid, dim3(kAttentionThreads), 0, s, a);
  else
    hipLaunchKernelGGL(prefix_attention_kernel<false>, grid, dim3(kAttentionThreads), 0, s, a);
  if (int32_t rc = check_launch("prefix_attention")) return rc;
  return launch_combine(*plan, a, workspace, s);
}
