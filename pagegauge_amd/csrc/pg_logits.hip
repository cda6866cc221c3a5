// Shaping of logits before a token is picked: penalties for the tokens of a
// request's history, biases, and a mask of allowed tokens.
//
//   x > 0 ? x / rep : x * rep      for tokens of the history
//   x - freq * c - pres * (c > 0)  c: occurrences since the prompt's end
//   x + bias
//   -inf                           where the mask's bit is clear
//
// One pass over the logits, in float32 with one rounding to their type.  A
// workgroup takes a tile of one row's vocabulary, counts the history's tokens
// that fall into it in LDS (integer atomics: the counts do not depend on the
// order), and applies everything as the logits pass through.  Each tile reads
// the whole history, which L2 serves to all tiles but the first; that is cheaper
// than counts of the whole vocabulary in memory, 4 bytes per logit and a
// launch to clear them.
#include "pg_common.h"

#include <hip/hip_bf16.h>

#include <algorithm>

namespace pg {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxTile = 8192;
constexpr int kMinTile = 1024;
constexpr uint32_t kSeen = 0x80000000u;    // in the history, made or not; low bits: times made
constexpr float kNegInf = -__builtin_huge_valf();

struct LogitsArgs {
  const void* logits;
  void* out;
  int64_t logits_stride, out_stride;
  int vocab, tile;
  const void* history;
  int64_t history_stride, history_capacity;
  const int32_t* history_lengths;
  const int32_t* prompt_lengths;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const void* bias_tokens;
  const float* bias_values;
  int biases;
  const int32_t* allowed;
  int64_t allowed_stride;
};

__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_float<__hip_bfloat16>(float v) {
  return __float2bfloat16(v);
}
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
  T v[kVec];
};

// Grid (tiles, rows); kVec 1 for rows that are not 16-byte aligned.
template <typename T, typename Token, int kVec>
__global__ __launch_bounds__(kThreads) void shape_logits_kernel(LogitsArgs a) {
  extern __shared__ uint32_t lds[];
  uint32_t* counts = lds;                                      // with a history
  int* bias_at = reinterpret_cast<int*>(lds) + (a.history ? a.tile : 0);   // with biases
  const int row = blockIdx.y;
  const int base = blockIdx.x * a.tile;
  const int size = min(a.tile, a.vocab - base);
  const int tid = threadIdx.x;
  if (a.history)
    for (int i = tid; i < a.tile; i += kThreads) counts[i] = 0u;
  if (a.biases)
    for (int i = tid; i < a.tile; i += kThreads) bias_at[i] = -1;
  __syncthreads();
  if (a.history) {
    const int64_t length = min(static_cast<int64_t>(a.history_lengths[row]), a.history_capacity);
    const int64_t prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    const Token* tokens = static_cast<const Token*>(a.history) + row * a.history_stride;
#pragma unroll 8
    for (int64_t i = tid; i < length; i += kThreads) {
      const int64_t at = static_cast<int64_t>(tokens[i]) - base;
      if (at < 0 || at >= size) continue;
      if (i >= prompt) atomicAdd(&counts[at], 1u); else atomicOr(&counts[at], kSeen);
    }
  }
  if (a.biases) {
    const Token* tokens = static_cast<const Token*>(a.bias_tokens) + static_cast<int64_t>(row) * a.biases;
    for (int i = tid; i < a.biases; i += kThreads) {
      const int64_t at = static_cast<int64_t>(tokens[i]) - base;
      if (at >= 0 && at < size) atomicMax(&bias_at[at], i);
    }
  }
  __syncthreads();
  const float repetition = a.repetition ? a.repetition[row] : 1.0f;
  const float frequency = a.frequency ? a.frequency[row] : 0.0f;
  const float presence = a.presence ? a.presence[row] : 0.0f;
  const float* bias_values = a.bias_values + static_cast<int64_t>(row) * a.biases;
  const int32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  auto shape = [&](float x, int at) {
    if (a.history) {
      const uint32_t c = counts[at];
      if (c) {
        if (a.repetition) x = x > 0.0f ? x / repetition : x * repetition;
        const uint32_t made = c & ~kSeen;
        if (made) {
          if (a.frequency) x -= frequency * static_cast<float>(made);
          if (a.presence) x -= presence;
        }
      }
    }
    if (a.biases) {
      const int b = bias_at[at];
      if (b >= 0) x += bias_values[b];
    }
    return x;
  };
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
  T* out = static_cast<T*>(a.out) + row * a.out_stride + base;
  for (int i = tid * kVec; i < size; i += kThreads * kVec) {
    // tiles and vectors are aligned to 32-token words of the mask
    const uint32_t word = allowed ? static_cast<uint32_t>(allowed[(base + i) >> 5]) >> (i & 31) : ~0u;
    if (kVec > 1 && i + kVec > size) {
      for (int e = 0; i + e < size; ++e)
        out[i + e] = word >> e & 1u ? from_float<T>(shape(to_float(in[i + e]), i + e)) : from_float<T>(kNegInf);
      break;
    }
    Vec<T, kVec> x = *reinterpret_cast<const Vec<T, kVec>*>(in + i);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      x.v[e] = word >> e & 1u ? from_float<T>(shape(to_float(x.v[e]), i + e)) : from_float<T>(kNegInf);
    *reinterpret_cast<Vec<T, kVec>*>(out + i) = x;
  }
}

template <typename T, typename Token>
int32_t launch(const LogitsArgs& a, int batch, bool wide, void* stream) {
  constexpr int kWide = 16 / sizeof(T);
  const dim3 grid((a.vocab + a.tile - 1) / a.tile, batch);
  const size_t lds = sizeof(uint32_t) * a.tile * ((a.history ? 1 : 0) + (a.biases ? 1 : 0));
  if (wide)
    hipLaunchKernelGGL((shape_logits_kernel<T, Token, kWide>), grid, dim3(kThreads), lds, as_stream(stream), a);
  else
    hipLaunchKernelGGL((shape_logits_kernel<T, Token, 1>), grid, dim3(kThreads), lds, as_stream(stream), a);
  return check_launch("shape_logits");
}

template <typename T>
int32_t dispatch(const LogitsArgs& a, int batch, int token_bytes, bool wide, void* stream) {
  return token_bytes == 8 ? launch<T, int64_t>(a, batch, wide, stream)
                          : launch<T, int32_t>(a, batch, wide, stream);
}

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_shape_logits(const void* logits, int64_t logits_stride, void* out,
                                   int64_t out_stride, int32_t dtype, int32_t batch, int32_t vocab,
                                   const void* history, int64_t history_stride,
                                   int64_t history_capacity, const int32_t* history_lengths,
                                   const int32_t* prompt_lengths, const float* repetition,
                                   const float* frequency, const float* presence,
                                   const void* bias_tokens, const float* bias_values, int32_t biases,
                                   int32_t token_bytes, const int32_t* allowed,
                                   int64_t allowed_stride, void* stream) {
  clear_error();
  if (!logits || !out) return fail(PG_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (batch < 0 || vocab <= 0) return fail(PG_ERROR_INVALID_ARGUMENT, "batch and vocabulary must be positive");
  if (batch > 65535) return fail(PG_ERROR_UNSUPPORTED, "at most 65535 rows of logits");
  if (vocab > 1 << 30) return fail(PG_ERROR_UNSUPPORTED, "at most 2^30 tokens of vocabulary");
  if (dtype < PG_DTYPE_FP16 || dtype > PG_DTYPE_FP32)
    return fail(PG_ERROR_INVALID_ARGUMENT, "logits must be FP16, BF16 or FP32");
  if (history && (!history_lengths || history_capacity < 0))
    return fail(PG_ERROR_INVALID_ARGUMENT, "a history needs its lengths");
  if (!history && (repetition || frequency || presence))
    return fail(PG_ERROR_INVALID_ARGUMENT, "penalties need a history");
  if (biases < 0 || (biases && (!bias_tokens || !bias_values)))
    return fail(PG_ERROR_INVALID_ARGUMENT, "bias tokens and values go together");
  if ((history || biases) && token_bytes != 4 && token_bytes != 8)
    return fail(PG_ERROR_INVALID_ARGUMENT, "tokens must be int32 or int64");
  if (batch == 0) return PG_OK;
  LogitsArgs a{};
  a.logits = logits;
  a.out = out;
  a.logits_stride = logits_stride;
  a.out_stride = out_stride;
  a.vocab = vocab;
  // tiles of 1024 to 8192 tokens, small ones where the batch leaves CUs idle
  a.tile = kMaxTile;
  while (a.tile > kMinTile && static_cast<int64_t>(batch) * ((vocab + a.tile - 1) / a.tile) < 512) a.tile /= 2;
  a.history = history && (repetition || frequency || presence) ? history : nullptr;
  a.history_stride = history_stride;
  a.history_capacity = history_capacity;
  a.history_lengths = history_lengths;
  a.prompt_lengths = prompt_lengths;
  a.repetition = repetition;
  a.frequency = frequency;
  a.presence = presence;
  a.bias_tokens = bias_tokens;
  a.bias_values = bias_values;
  a.biases = biases;
  a.allowed = allowed;
  a.allowed_stride = allowed_stride;
  const int64_t size = dtype == PG_DTYPE_FP32 ? 4 : 2;
  const bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                    (logits_stride * size) % 16 == 0 && (out_stride * size) % 16 == 0;
  switch (dtype) {
    case PG_DTYPE_FP16: return dispatch<__half>(a, batch, token_bytes, wide, stream);
    case PG_DTYPE_BF16: return dispatch<__hip_bfloat16>(a, batch, token_bytes, wide, stream);
    default: return dispatch<float>(a, batch, token_bytes, wide, stream);
  }
}
