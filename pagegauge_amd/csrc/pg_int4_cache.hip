// Writers and reader-back of the cache held in 4 bits (layout: pg_int4.h).
//
// A token's row x (128 dims of a KV head, K or V, minus the request's channel
// center) is held as code * scale:
//   scale = fp16(max(max|x| * (1/7), 2^-20)),
//   code  = sign(x) floor(|x / scale| + 0.5) clamped to [-7, 7], a NaN giving 0,
// in float32, 1/7 rounded to it and the quotient IEEE's: the INT8 pages' finalize
// with 7 steps for 127, and a product for its division by the steps.  A scale
// per token and head costs 1/32 of the codes and keeps an outlying token
// to itself; a scale per page would share it with 15 others.
//
// One wave takes one K or V part of a block and holds it in registers in the
// lane order of the packed layout, so that codes leave as one 1 KiB store of 16
// bytes per lane.  All kernels are bound by HBM once they fill the chip, by a trip
// or two to it before.  16384 tokens of 8 heads: quantized (84 MB) in 21.3 us and read
// back in 21.1, rows from and to HBM, where a copy of as many bytes takes 17.4 (19.4
// and 16.2 where the Infinity Cache holds the rows); 1000 tokens 4.3 us each.  The
// quantizer's arithmetic is what is left of its distance: 32.5 us with a division per
// code, 25.3 with clamps and selects.  Reading back took 23.8 with conversions of
// integers and half lines per store.
#include "pg_int4.h"
#include "pg_rotary.h"

#include <algorithm>

namespace pg {
namespace {

typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kWavesPerBlock = 4;
constexpr int64_t kMaxBlocks = UINT32_MAX / (kWave * kWavesPerBlock);   // of a launch's first dimension

__device__ __forceinline__ uint16_t int4_scale_bits(float maximum) {
  return __half_as_ushort(__float2half_rn(fmaxf(maximum * (1.0f / 7.0f), 0x1p-20f)));
}

// Code of x / scale, given r = 1 / scale to an ulp: the quotient is the IEEE one,
// by three operations instead of a division.  q0 = RN(x * r) is within 3 ulp of
// it, the residual e = x - q0 * scale is exact (the scale has the 11 bits of an
// FP16 value, so e has 13; x lies far from float32's limits), and q0 + e * r is
// the quotient to 2^-20 ulp before it is rounded; a 24-bit number over an 11-bit
// one is never within 2^-12 ulp of a midpoint of two floats.  An infinite scale
// gives NaN for every x where the division gives 0 or NaN, and both have code 0.
//
// sign(q) floor(|q| + 0.5) is the truncation of q + copysign(0.5, q).  No clamp
// is needed: a stored scale is at least (1 - 2^-5) max|x| / 7 (2^-20 is a subnormal
// FP16 number), so |q| < 7.25.  The conversion instruction takes a NaN to 0 (C++
// leaves that open).
__device__ __forceinline__ int int4_code(float x, float scale, float r) {
  const float q0 = x * r;
  const float q = fmaf(fmaf(-q0, scale, x), r, q0);
  int code;
  asm("v_cvt_i32_f32 %0, %1" : "=v"(code) : "v"(q + __builtin_copysignf(0.5f, q)));
  return code;
}

// Eight nibbles, code + 8 each, start at 8 8 ... 8; adding a code at its place
// never carries out of it.
constexpr uint32_t kNibbles8 = 0x88888888u;
__device__ __forceinline__ uint32_t put_code(uint32_t word, int code, int nibble) {
  return word + (static_cast<uint32_t>(code) << (4 * nibble));
}

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// Value e of eight minus center e, rounded to float32: one mixed-precision
// operation (``one`` is 1, where the compiler does not see it).
__device__ __forceinline__ float centered_at(const v4u& v, const v4u& c, int e, float one) {
  return fmaf(static_cast<float>(__builtin_bit_cast(v8h, v)[e]), one,
              -static_cast<float>(__builtin_bit_cast(v8h, c)[e]));
}

__device__ __forceinline__ float half_at(const v4u& v, int e) {
  return half_bits_to_float(static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1))));
}

// Eight FP16 values at ``p``, which need only be aligned to 2 bytes unless kWide.
template <bool kWide>
__device__ __forceinline__ v4u load8(const uint16_t* p) {
  if (kWide) return *reinterpret_cast<const v4u*>(p);
  v4u v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
  return v;
}

template <bool kWide>
__device__ __forceinline__ void store8(uint16_t* p, const v4u& v) {
  if (kWide) {
    *reinterpret_cast<v4u*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[2 * i] = static_cast<uint16_t>(v[i]);
    p[2 * i + 1] = static_cast<uint16_t>(v[i] >> 16);
  }
}

// Packs one part from the wave's registers: x[g][e] is dim 32 g + 8 kg + e of
// token n (K), or channel 8 n + e of token 4 kg + g (V).  Rows at or past
// ``visible`` are stored as scale 0.
template <bool kValue>
__device__ __forceinline__ void pack_part(const float (&x)[4][8], int visible, uint8_t* codes,
                                          uint16_t* scales, int lane) {
  const int n = lane & 15, kg = lane >> 4;
  v4u word = {kNibbles8, kNibbles8, kNibbles8, kNibbles8};
  if (!kValue) {
    float m = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[g][e]));
    m = fmaxf(m, __shfl_xor(m, 16, kWave));
    m = fmaxf(m, __shfl_xor(m, 32, kWave));
    const uint16_t bits = int4_scale_bits(m);
    const float scale = half_bits_to_float(bits), r = __builtin_amdgcn_rcpf(scale);
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        word[g] = put_code(word[g], int4_code(x[g][e], scale, r), (e >> 1) + 4 * (e & 1));
    if (kg == 0) scales[int4_scale_index(0, n)] = n < visible ? bits : 0;
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[t][e]));
      const uint16_t bits = int4_scale_bits(row16_max(m));
      const float scale = half_bits_to_float(bits), r = __builtin_amdgcn_rcpf(scale);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        word[e >> 1] = put_code(word[e >> 1], int4_code(x[t][e], scale, r), (t >> 1) + 2 * (e & 1) + 4 * (t & 1));
      if (n == 0) scales[int4_scale_index(1, 4 * kg + t)] = 4 * kg + t < visible ? bits : 0;
    }
  }
  *reinterpret_cast<v4u*>(codes + 16 * lane) = word;
}

// The row of part registers x[g] and its first dim, of the lane order above.
template <bool kValue>
__device__ __forceinline__ int part_row(int g, int lane) {
  return kValue ? 4 * (lane >> 4) + g : lane & 15;
}
template <bool kValue>
__device__ __forceinline__ int part_dim(int g, int lane) {
  return kValue ? 8 * (lane & 15) : 32 * g + 8 * (lane >> 4);
}

struct QuantizeArgs {
  const uint16_t* source[2];       // token-major K and V rows
  int64_t token_stride[2];
  const uint16_t* center[2];       // [Hkv, 128] or null
  uint8_t* codes;
  uint16_t* scales;
  const int32_t* page_ids;         // code page of each source page, or null: the same
  const int32_t* exact_ids;        // exact page of each source page, or null
  uint16_t* exact[2];
  int64_t tokens, pages, num_code_pages, num_exact_pages;
  int heads;
};

template <bool kWide, bool kValue>
__device__ __forceinline__ void quantize_part(const QuantizeArgs& a, int64_t page, int head, int lane) {
  const int64_t code_page = a.page_ids ? a.page_ids[page] : page;
  const int64_t exact_page = a.exact_ids ? a.exact_ids[page] : -1;
  const int visible = static_cast<int>(min(static_cast<int64_t>(kPageSize), a.tokens - page * kPageSize));
  const uint16_t* source = a.source[kValue] + page * kPageSize * a.token_stride[kValue] + head * kHeadDim;
  const uint16_t* center = a.center[kValue];
  float x[4][8];
  v4u raw[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int row = part_row<kValue>(g, lane);
    const int64_t at = min(row, visible - 1) * a.token_stride[kValue] + part_dim<kValue>(g, lane);
    raw[g] = load8<kWide>(source + at);
  }
  float one = 1.0f;
  asm("" : "+v"(one));
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    v4u c = {0u, 0u, 0u, 0u};
    if (center) c = load8<kWide>(center + head * kHeadDim + part_dim<kValue>(g, lane));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[g][e] = centered_at(raw[g], c, e, one);
  }
  if (visible < kPageSize) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[g][e] = part_row<kValue>(g, lane) < visible ? x[g][e] : 0.0f;
  }
  if (exact_page >= 0 && exact_page < a.num_exact_pages) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int row = part_row<kValue>(g, lane);
      if (row >= visible) continue;
      v4u out;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[i] = __half_as_ushort(__float2half_rn(x[g][2 * i])) |
                 static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[g][2 * i + 1]))) << 16;
      store8<kWide>(a.exact[kValue] + ((exact_page * kPageSize + row) * a.heads + head) * kHeadDim +
                        part_dim<kValue>(g, lane), out);
    }
  }
  if (code_page < 0 || code_page >= a.num_code_pages) return;
  const int64_t block = code_page * a.heads + head;
  pack_part<kValue>(x, visible, a.codes + block * kInt4BlockBytes + kValue * kInt4PartBytes,
                    a.scales + block * kInt4BlockScales, lane);
}

// A wave per (page, head), in the order of memory: blocks of up to 4 heads of page
// after page by blockIdx.x, K and V by blockIdx.y.
template <bool kWide>
__global__ __launch_bounds__(kWave * kWavesPerBlock) void int4_quantize_kernel(QuantizeArgs a) {
  const int waves = blockDim.x / kWave, per_page = (a.heads + waves - 1) / waves;
  const int64_t page = blockIdx.x / per_page;
  const int head = blockIdx.x % per_page * waves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (head >= a.heads) return;
  if (blockIdx.y == 0)
    quantize_part<kWide, false>(a, page, head, threadIdx.x % kWave);
  else
    quantize_part<kWide, true>(a, page, head, threadIdx.x % kWave);
}

struct DequantizeArgs {
  const uint8_t* codes;
  const uint16_t* scales;
  const int32_t* page_ids;
  const uint16_t* center[2];
  uint16_t* out[2];
  int64_t token_stride[2];
  int64_t tokens, pages, num_code_pages;
  int heads;
};

// Lane n's word from lane n ^ 8 of the same 16.
__device__ __forceinline__ uint32_t across8(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x128 /* row_ror:8 */, 0xf, 0xf, false);
}

// Codes in nibbles i and i + 4 of a word: a masked nibble is the FP16 subnormal
// u * 2^-24, or 16 u * 2^-24 one nibble further up, and less 8 of the same it is the
// code, exactly.
__device__ __forceinline__ v2h code_pair(uint32_t word, int i) {
  const uint32_t shifted = i & 2 ? word >> 8 : word;
  const uint32_t bits = shifted & (i & 1 ? 0x00f000f0u : 0x000f000fu);
  return __builtin_bit_cast(v2h, bits) - __builtin_bit_cast(v2h, i & 1 ? 0x00800080u : 0x00080008u);
}

// Rounded to float32, then to FP16, as the formula is.
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
  return __half_as_ushort(__float2half_rn(a)) | static_cast<uint32_t>(__half_as_ushort(__float2half_rn(b))) << 16;
}

template <bool kWide, bool kValue>
__device__ __forceinline__ void dequantize_part(const DequantizeArgs& a, int64_t page, int head, int lane) {
  const int64_t code_page = a.page_ids ? a.page_ids[page] : page;
  const int64_t visible = a.tokens - page * kPageSize;
  const bool held = code_page >= 0 && code_page < a.num_code_pages;
  const int64_t block = (held ? code_page : 0) * a.heads + head;
  const uint16_t* scales = a.scales + block * kInt4BlockScales;
  v4u word = *reinterpret_cast<const v4u*>(a.codes + block * kInt4BlockBytes +
                                           kValue * kInt4PartBytes + 16 * lane);
  const bool upper = lane & 8;
  // row and dim of store g: V's are those of the lane; K's lanes n and n + 8 trade
  // words, so that a store writes whole lines: words 2 j and 2 j + 1 of lane n become
  // dims 64 j + 32 (n / 8) .. of tokens n % 8 and n % 8 + 8 (half lines of 16 tokens
  // per store took 23.2 us where this took 21.8)
  auto row_of = [&](int g) { return kValue ? part_row<true>(g, lane) : (lane & 7) + 8 * (g & 1); };
  auto dim_of = [&](int g) {
    return kValue ? part_dim<true>(g, lane) : 64 * (g >> 1) + 32 * upper + 8 * (lane >> 4);
  };
  if (!kValue) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const uint32_t other = across8(upper ? word[j] : word[j + 1]);
      word[j] = upper ? other : word[j];
      word[j + 1] = upper ? word[j + 1] : other;
    }
  }
  float scale[4];
  v8h center[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    scale[g] = held ? half_bits_to_float(scales[int4_scale_index(kValue, row_of(g))]) : 0.0f;
    v4u c = {0u, 0u, 0u, 0u};
    if (a.center[kValue] && held) c = load8<kWide>(a.center[kValue] + head * kHeadDim + dim_of(g));
    center[g] = __builtin_bit_cast(v8h, c);
  }
  auto value = [&](v2h codes, int half, int i, int g, int e) {
    return fmaf(static_cast<float>(codes[half]), scale[g] * (i & 1 ? 0x1p20f : 0x1p24f),
                static_cast<float>(center[g][e]));
  };
  v4u out[4];
  if (!kValue) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // dims 2 i and 2 i + 1
        const v2h codes = code_pair(word[g], i);
        out[g][i] = half_pair(value(codes, 0, i, g, 2 * i), value(codes, 1, i, g, 2 * i + 1));
      }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < 4; t += 2) {   // tokens t and t + 1, channels 2 j and 2 j + 1
        const int i = t >> 1;
        const v2h even = code_pair(word[j], i), odd = code_pair(word[j], i + 2);
        out[t][j] = half_pair(value(even, 0, i, t, 2 * j), value(odd, 0, i, t, 2 * j + 1));
        out[t + 1][j] = half_pair(value(even, 1, i, t + 1, 2 * j), value(odd, 1, i, t + 1, 2 * j + 1));
      }
  }
  uint16_t* rows = a.out[kValue] + page * kPageSize * a.token_stride[kValue] + head * kHeadDim;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (row_of(g) < visible) store8<kWide>(rows + row_of(g) * a.token_stride[kValue] + dim_of(g), out[g]);
}

template <bool kWide>
__global__ __launch_bounds__(kWave * kWavesPerBlock) void int4_dequantize_kernel(DequantizeArgs a) {
  const int waves = blockDim.x / kWave, per_page = (a.heads + waves - 1) / waves;
  const int64_t page = blockIdx.x / per_page;
  const int head = blockIdx.x % per_page * waves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (head >= a.heads) return;
  if (blockIdx.y == 0)
    dequantize_part<kWide, false>(a, page, head, threadIdx.x % kWave);
  else
    dequantize_part<kWide, true>(a, page, head, threadIdx.x % kWave);
}

struct AppendArgs {
  const uint16_t* rows[3];         // query, key, value [B, H, 128]
  int64_t batch_stride[3];
  uint16_t* rotated_query;
  const int32_t* positions;
  const double* turns;
  float amplitude;
  int rotary_dim, interleaved;
  const int32_t* exact_ids;
  const int32_t* code_ids;
  const uint16_t* center[2];       // [B, Hkv, 128]
  uint16_t* exact[2];
  uint8_t* codes;
  uint16_t* scales;
  int64_t num_exact_pages, num_code_pages;
  int query_heads, kv_heads;
};

constexpr int kQueryRows = 4;      // query heads of a wave

// One wave per 4 query heads of a request, then per K and per V head: lane p
// holds pair p of the rotated part, or two dims past it.  What the rows need is
// requested at once, the rows of a page that closes included: the kernel's time
// is that of its trips to memory, one for the request's position and ids and one
// for everything else (as a chain of five, 256 requests took 10.4 us in place of
// 6.9).  With a wave per query head, more than the chip holds at once, 256 requests
// of 32 query and 8 KV heads took 6.9 us and 1024 took 15.0; now 6.3 to 7.4 and 11.2, and
// 3.7 to 4.4 for 8 requests that all close a page.  Large batches are bound by its accesses
// of 2 bytes per lane and the sines that 16 waves of a request work out alike: at a copy's
// rate their bytes take 1.7 and 6.7 us (5.5 and 22 where all close a page, now 8.7 and 23.8).
__global__ __launch_bounds__(kWave * kWavesPerBlock) void int4_rope_append_kernel(AppendArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t own[kWavesPerBlock][kHeadDim];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int row = blockIdx.y * kWavesPerBlock + wave;
  const int query_waves = (a.query_heads + kQueryRows - 1) / kQueryRows;
  if (row >= query_waves + 2 * a.kv_heads) return;     // whole waves; no barrier below
  const int request = blockIdx.x;
  const bool turned = lane < a.rotary_dim / 2;
  const int first = turned && !a.interleaved ? lane : 2 * lane;
  const int second = turned && !a.interleaved ? lane + a.rotary_dim / 2 : 2 * lane + 1;
  if (row < query_waves) {
    const int head = row * kQueryRows, heads = min(kQueryRows, a.query_heads - head);
    const uint16_t* in = a.rows[0] + request * a.batch_stride[0] + head * kHeadDim;
    uint16_t x_bits[kQueryRows], y_bits[kQueryRows];
#pragma unroll
    for (int k = 0; k < kQueryRows; ++k) {
      x_bits[k] = in[min(k, heads - 1) * kHeadDim + first];
      y_bits[k] = in[min(k, heads - 1) * kHeadDim + second];
    }
    const double turns = a.turns[turned ? lane : 0];
    const int32_t position = a.positions[request];
    if (position < 0) return;
    const float2 cos_sin = rotary_cos_sin(position, turns, a.amplitude);
    uint16_t* out = a.rotated_query + (static_cast<int64_t>(request) * a.query_heads + head) * kHeadDim;
#pragma unroll
    for (int k = 0; k < kQueryRows; ++k) {
      if (k >= heads) break;
      const float2 pair = rotate_pair(half_bits_to_float(x_bits[k]), half_bits_to_float(y_bits[k]), cos_sin);
      out[k * kHeadDim + first] = turned ? __half_as_ushort(__float2half_rn(pair.x)) : x_bits[k];
      out[k * kHeadDim + second] = turned ? __half_as_ushort(__float2half_rn(pair.y)) : y_bits[k];
    }
    return;
  }
  const int kind = row < query_waves + a.kv_heads ? 1 : 2;
  const int head = row - query_waves - (kind == 1 ? 0 : a.kv_heads);
  const uint16_t* in = a.rows[kind] + request * a.batch_stride[kind] + head * kHeadDim;
  const int32_t position = a.positions[request];
  const int64_t exact_page = a.exact_ids[request], code_page = a.code_ids[request];
  const uint16_t x_bits = in[first], y_bits = in[second];
  const double turns = a.turns[turned ? lane : 0];
  if (position < 0) return;
  const int offset = position % kPageSize;
  if (exact_page < 0 || exact_page >= a.num_exact_pages) return;
  const bool closes = offset == kPageSize - 1 && code_page >= 0 && code_page < a.num_code_pages;

  // rows of the page in the packed order; row 15 is this token's own and comes
  // from LDS, row 14 is read in its place
  v4u held[4];
  const int64_t row_stride = static_cast<int64_t>(a.kv_heads) * kHeadDim;
  uint16_t* page = a.exact[kind - 1] + exact_page * kPageSize * row_stride + head * kHeadDim;
  if (closes) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = kind == 1 ? part_row<false>(g, lane) : part_row<true>(g, lane);
      const int dim = kind == 1 ? part_dim<false>(g, lane) : part_dim<true>(g, lane);
      held[g] = *reinterpret_cast<const v4u*>(page + min(r, kPageSize - 2) * row_stride + dim);
    }
  }
  const uint16_t* center = a.center[kind - 1] + (static_cast<int64_t>(request) * a.kv_heads + head) * kHeadDim;
  const float cx = half_bits_to_float(center[first]), cy = half_bits_to_float(center[second]);
  float x = half_bits_to_float(x_bits), y = half_bits_to_float(y_bits);
  if (kind == 1 && turned) {
    const float2 pair = rotate_pair(x, y, rotary_cos_sin(position, turns, a.amplitude));
    x = pair.x;
    y = pair.y;
  }
  const uint16_t xb = __half_as_ushort(__float2half_rn(x - cx));
  const uint16_t yb = __half_as_ushort(__float2half_rn(y - cy));
  page[offset * row_stride + first] = xb;
  page[offset * row_stride + second] = yb;
  if (!closes) return;
  own[wave][first] = xb;
  own[wave][second] = yb;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int64_t block = code_page * a.kv_heads + head;
  uint8_t* codes = a.codes + block * kInt4BlockBytes;
  uint16_t* scales = a.scales + block * kInt4BlockScales;
  float rows[4][8];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int r = kind == 1 ? part_row<false>(g, lane) : part_row<true>(g, lane);
    const int dim = kind == 1 ? part_dim<false>(g, lane) : part_dim<true>(g, lane);
    const v4u mine = *reinterpret_cast<const v4u*>(own[wave] + dim);
    const v4u raw = r == kPageSize - 1 ? mine : held[g];
#pragma unroll
    for (int e = 0; e < 8; ++e) rows[g][e] = half_at(raw, e);
  }
  if (kind == 1)
    pack_part<false>(rows, kPageSize, codes, scales, lane);
  else
    pack_part<true>(rows, kPageSize, codes + kInt4PartBytes, scales, lane);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int32_t check_pool(const void* codes, const void* scales, int64_t num_code_pages, int32_t heads) {
  if (!codes || !scales) return fail(PG_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned16(codes) || !aligned16(scales))
    return fail(PG_ERROR_INVALID_ARGUMENT, "4-bit codes and scales must be 16-byte aligned");
  if (num_code_pages < 0 || heads <= 0)
    return fail(PG_ERROR_INVALID_ARGUMENT, "page and head counts must be positive");
  if (heads > 65535) return fail(PG_ERROR_UNSUPPORTED, "at most 65535 KV heads");
  return PG_OK;
}

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_int4_quantize_pages(const void* key, int64_t key_token_stride, const void* value,
                                          int64_t value_token_stride, const void* key_center,
                                          const void* value_center, void* codes, void* scales,
                                          int64_t num_code_pages, const int32_t* page_ids,
                                          const int32_t* exact_page_ids, void* exact_key_pages,
                                          void* exact_value_pages, int64_t num_exact_pages,
                                          int64_t tokens, int32_t heads, void* stream) {
  clear_error();
  if (!key || !value) return fail(PG_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (int32_t rc = check_pool(codes, scales, num_code_pages, heads)) return rc;
  if ((key_center == nullptr) != (value_center == nullptr))
    return fail(PG_ERROR_INVALID_ARGUMENT, "key and value centers go together");
  if (exact_page_ids && (!exact_key_pages || !exact_value_pages || num_exact_pages < 0))
    return fail(PG_ERROR_INVALID_ARGUMENT, "exact page ids need exact key/value pages");
  if (tokens < 0) return fail(PG_ERROR_INVALID_ARGUMENT, "token count must be nonnegative");
  if (tokens == 0) return PG_OK;
  QuantizeArgs a{};
  a.source[0] = static_cast<const uint16_t*>(key);
  a.source[1] = static_cast<const uint16_t*>(value);
  a.token_stride[0] = key_token_stride;
  a.token_stride[1] = value_token_stride;
  a.center[0] = static_cast<const uint16_t*>(key_center);
  a.center[1] = static_cast<const uint16_t*>(value_center);
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint16_t*>(scales);
  a.page_ids = page_ids;
  a.exact_ids = exact_page_ids;
  a.exact[0] = static_cast<uint16_t*>(exact_key_pages);
  a.exact[1] = static_cast<uint16_t*>(exact_value_pages);
  a.tokens = tokens;
  a.pages = (tokens - 1) / kPageSize + 1;
  a.num_code_pages = num_code_pages;
  a.num_exact_pages = exact_page_ids ? num_exact_pages : 0;
  a.heads = heads;
  bool wide = key_token_stride % 8 == 0 && value_token_stride % 8 == 0;
  for (const void* p : {key, value, key_center, value_center,
                        static_cast<const void*>(exact_key_pages), static_cast<const void*>(exact_value_pages)})
    wide = wide && aligned16(p);
  const int waves = std::min(heads, kWavesPerBlock), per_page = (heads + waves - 1) / waves;
  if (a.pages > kMaxBlocks / per_page) return fail(PG_ERROR_UNSUPPORTED, "too many pages for one call");
  const dim3 grid(static_cast<uint32_t>(a.pages * per_page), 2);
  if (wide)
    hipLaunchKernelGGL(int4_quantize_kernel<true>, grid, dim3(kWave * waves), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(int4_quantize_kernel<false>, grid, dim3(kWave * waves), 0, as_stream(stream), a);
  return check_launch("int4_quantize_pages");
}

extern "C" int32_t pg_int4_dequantize_pages(const void* codes, const void* scales,
                                            int64_t num_code_pages, const int32_t* page_ids,
                                            const void* key_center, const void* value_center,
                                            void* key, int64_t key_token_stride, void* value,
                                            int64_t value_token_stride, int64_t tokens,
                                            int32_t heads, void* stream) {
  clear_error();
  if (!key || !value) return fail(PG_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (int32_t rc = check_pool(codes, scales, num_code_pages, heads)) return rc;
  if ((key_center == nullptr) != (value_center == nullptr))
    return fail(PG_ERROR_INVALID_ARGUMENT, "key and value centers go together");
  if (tokens < 0) return fail(PG_ERROR_INVALID_ARGUMENT, "token count must be nonnegative");
  if (tokens == 0) return PG_OK;
  if (num_code_pages == 0) return fail(PG_ERROR_INVALID_ARGUMENT, "the pool holds no pages");
  DequantizeArgs a{};
  a.codes = static_cast<const uint8_t*>(codes);
  a.scales = static_cast<const uint16_t*>(scales);
  a.page_ids = page_ids;
  a.center[0] = static_cast<const uint16_t*>(key_center);
  a.center[1] = static_cast<const uint16_t*>(value_center);
  a.out[0] = static_cast<uint16_t*>(key);
  a.out[1] = static_cast<uint16_t*>(value);
  a.token_stride[0] = key_token_stride;
  a.token_stride[1] = value_token_stride;
  a.tokens = tokens;
  a.pages = (tokens - 1) / kPageSize + 1;
  a.num_code_pages = num_code_pages;
  a.heads = heads;
  bool wide = key_token_stride % 8 == 0 && value_token_stride % 8 == 0;
  for (const void* p : {key_center, value_center, static_cast<const void*>(key), static_cast<const void*>(value)})
    wide = wide && aligned16(p);
  const int waves = std::min(heads, kWavesPerBlock), per_page = (heads + waves - 1) / waves;
  if (a.pages > kMaxBlocks / per_page) return fail(PG_ERROR_UNSUPPORTED, "too many pages for one call");
  const dim3 grid(static_cast<uint32_t>(a.pages * per_page), 2);
  if (wide)
    hipLaunchKernelGGL(int4_dequantize_kernel<true>, grid, dim3(kWave * waves), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(int4_dequantize_kernel<false>, grid, dim3(kWave * waves), 0, as_stream(stream), a);
  return check_launch("int4_dequantize_pages");
}

extern "C" int32_t pg_int4_rope_append(
    const void* query, const void* key, const void* value, int64_t query_batch_stride,
    int64_t key_batch_stride, int64_t value_batch_stride, const int32_t* positions,
    const double* turns, float amplitude, int32_t rotary_dim, int32_t interleaved,
    const int32_t* exact_page_ids, const int32_t* code_page_ids, const void* key_center,
    const void* value_center, void* rotated_query, void* exact_key_pages, void* exact_value_pages,
    int64_t num_exact_pages, void* codes, void* scales, int64_t num_code_pages,
    int32_t batch_size, int32_t query_heads, int32_t kv_heads, void* stream) {
  clear_error();
  if (!query || !key || !value || !positions || !turns || !exact_page_ids || !code_page_ids ||
      !key_center || !value_center || !rotated_query || !exact_key_pages || !exact_value_pages)
    return fail(PG_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (int32_t rc = check_pool(codes, scales, num_code_pages, kv_heads)) return rc;
  if (!aligned16(exact_key_pages) || !aligned16(exact_value_pages))
    return fail(PG_ERROR_INVALID_ARGUMENT, "exact pages must be 16-byte aligned");
  if (batch_size < 0 || num_exact_pages < 0 || query_heads <= 0)
    return fail(PG_ERROR_INVALID_ARGUMENT, "batch, head and page counts must be positive");
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > kHeadDim)
    return fail(PG_ERROR_INVALID_ARGUMENT, "the rotated part must be an even number of a head's dims");
  const int64_t query_waves = (static_cast<int64_t>(query_heads) + kQueryRows - 1) / kQueryRows;
  const int64_t row_blocks = (query_waves + 2 * kv_heads + kWavesPerBlock - 1) / kWavesPerBlock;
  if (row_blocks > 65535) return fail(PG_ERROR_UNSUPPORTED, "too many heads for one call");
  if (batch_size > kMaxBlocks) return fail(PG_ERROR_UNSUPPORTED, "too many requests for one call");
  if (batch_size == 0) return PG_OK;
  AppendArgs a{};
  a.rows[0] = static_cast<const uint16_t*>(query);
  a.rows[1] = static_cast<const uint16_t*>(key);
  a.rows[2] = static_cast<const uint16_t*>(value);
  a.batch_stride[0] = query_batch_stride;
  a.batch_stride[1] = key_batch_stride;
  a.batch_stride[2] = value_batch_stride;
  a.rotated_query = static_cast<uint16_t*>(rotated_query);
  a.positions = positions;
  a.turns = turns;
  a.amplitude = amplitude;
  a.rotary_dim = rotary_dim;
  a.interleaved = interleaved;
  a.exact_ids = exact_page_ids;
  a.code_ids = code_page_ids;
  a.center[0] = static_cast<const uint16_t*>(key_center);
  a.center[1] = static_cast<const uint16_t*>(value_center);
  a.exact[0] = static_cast<uint16_t*>(exact_key_pages);
  a.exact[1] = static_cast<uint16_t*>(exact_value_pages);
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint16_t*>(scales);
  a.num_exact_pages = num_exact_pages;
  a.num_code_pages = num_code_pages;
  a.query_heads = query_heads;
  a.kv_heads = kv_heads;
  hipLaunchKernelGGL(int4_rope_append_kernel, dim3(batch_size, static_cast<uint32_t>(row_blocks)),
                     dim3(kWave * kWavesPerBlock), 0, as_stream(stream), a);
  return check_launch("int4_rope_append");
}
