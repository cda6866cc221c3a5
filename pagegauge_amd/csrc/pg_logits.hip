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
//
// Bound by HBM and, in turn, by the steps before the logits can leave: 64 rows of
// 131072 float32 logits (70 MB) with histories of 4096, 64 biases and a mask take
// 16.6 to 17.4 us, where a copy of as many bytes takes 13.5.  Of these the mask
// costs 2, cleared counts and barriers 1.7, the histories 3.5 and the biases 0.5
// to 1.  One row of 32768 takes 5.6 us.  Measured and not taken at 64 rows: 512
// threads with tiles of 4096 or 8192 (19.5, 20.5 us), 256 with 4096 (22.3), and
// two tiles per workgroup with the tokens kept in registers (21.2).
#include "pg_types.h"

#include <algorithm>

namespace pg {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxTile = 8192;
constexpr int kMinTile = 1024;
// a token's count: times made, and whether the history or the biases have it
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u;
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

// Grid (rows, tiles), so that the tiles of a row are a multiple of the batch apart
// and, in batches of whole eights, share an XCD's L2 for the row's history (64 rows
// 17.2 us, tiles first 17.8).  With kVec 1 a value at a time; kShifted for rows that do
// not all start with a vector: a tile's index 0 does, and a row starts ``pad`` values
// into its first tile (51 rows of 103354 12.1 us, a value at a time 16.2).
//
// The tile's logits and the first tokens of the history are requested before
// anything else, so that the trips to memory overlap (64 x 131072 with
// histories of 4096: 20.5 us one after the other).
template <typename T, typename Token, int kVec, bool kShifted>
__global__ __launch_bounds__(kThreads) void shape_logits_kernel(LogitsArgs a) {
  constexpr int kSteps = kVec > 1 ? kMaxTile / (kThreads * kVec) : 1;
  constexpr int kBatch = 4;                                    // tokens of a thread in flight
  extern __shared__ uint32_t lds[];
  uint32_t* counts = lds;
  int* bias_at = reinterpret_cast<int*>(lds) + a.tile;         // of the tokens that have a bias
  const int row = blockIdx.x;
  const int tid = threadIdx.x;
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  T* out = static_cast<T*>(a.out) + row * a.out_stride;
  const int pad = kShifted ? reinterpret_cast<uintptr_t>(in) / sizeof(T) % kVec : 0;
  const int base = static_cast<int>(blockIdx.y) * a.tile - pad;      // token at index 0
  const int low = kShifted && base < 0 ? pad : 0, size = min(a.tile, a.vocab - base);   // the tile's tokens
  in += base;
  out += base;
  if (kShifted && low >= size) return;       // the last tile of a row that needs none
  const int32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  // the mask's bits of the tokens from index i on, of the kVec of a vector with ``both``
  auto bits = [&](int i, bool both) {
    if (!allowed) return ~0u;
    const int token = base + i;
    const uint32_t word = allowed[token >> 5];
    if (!kShifted || !both) return word >> (token & 31);
    const uint64_t next = static_cast<uint32_t>(allowed[(token + kVec - 1) >> 5]);
    return static_cast<uint32_t>((next << 32 | word) >> (token & 31));
  };
  // whole vectors [whole, rest), and a thread for each value before and behind them;
  // with kVec 1 a thread for each of the first kThreads
  const int whole = (low + kVec - 1) / kVec * kVec, rest = max(whole, size / kVec * kVec);
  const int edge = kVec == 1 || tid < kVec ? low + tid : rest + tid - kVec;
  const bool has_edge = kVec == 1 ? edge < size
                                  : tid < 2 * kVec && edge < (tid < kVec ? min(whole, size) : size);
  Vec<T, kVec> held[kSteps];
  uint32_t words[kSteps];
  if (kVec > 1 && whole < rest) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      // where there is no whole vector, the first one is read and not used
      const int i = (tid + s * kThreads) * kVec, at = i >= whole && i < rest ? i : whole;
      held[s] = *reinterpret_cast<const Vec<T, kVec>*>(in + at);
      words[s] = bits(at, true);
    }
  }
  T edge_value{};
  uint32_t edge_bits = 0;
  if (has_edge) {
    edge_value = in[edge];
    edge_bits = bits(edge, false);
  }
  const float repetition = a.repetition ? a.repetition[row] : 1.0f;
  const float frequency = a.frequency ? a.frequency[row] : 0.0f;
  const float presence = a.presence ? a.presence[row] : 0.0f;
  const bool counted = a.history || a.biases;
  const Token* tokens = static_cast<const Token*>(a.history) + row * a.history_stride;
  int64_t length = 0, prompt = 0;
  Token batch[kBatch];
  auto request_tokens = [&](int64_t first) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int64_t i = first + tid + k * kThreads;
      batch[k] = tokens[i < length ? i : length - 1];
    }
  };
  if (a.history) {
    length = max(int64_t{0}, min(static_cast<int64_t>(a.history_lengths[row]), a.history_capacity));
    if (a.prompt_lengths) prompt = a.prompt_lengths[row];
    if (length > 0) request_tokens(0);
  }
  const Token* bias_tokens = static_cast<const Token*>(a.bias_tokens) + static_cast<int64_t>(row) * a.biases;
  if (counted) {
    for (int i = tid; i < a.tile / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = uint4{0u, 0u, 0u, 0u};
    for (int i = tid; i < a.biases; i += kThreads) {
      const int64_t at = static_cast<int64_t>(bias_tokens[i]) - base;
      if (at >= low && at < size) bias_at[at] = -1;
    }
    __syncthreads();
    for (int64_t first = 0; first < length; first += kBatch * kThreads) {
      if (first) request_tokens(first);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int64_t i = first + tid + k * kThreads;
        const int64_t at = static_cast<int64_t>(batch[k]) - base;
        if (i >= length || at < low || at >= size) continue;
        if (i >= prompt) atomicAdd(&counts[at], 1u); else atomicOr(&counts[at], kSeen);
      }
    }
    for (int i = tid; i < a.biases; i += kThreads) {
      const int64_t at = static_cast<int64_t>(bias_tokens[i]) - base;
      if (at < low || at >= size) continue;
      atomicMax(&bias_at[at], i);
      atomicOr(&counts[at], kBiased);
    }
    __syncthreads();
  }
  const float* bias_values = a.bias_values + static_cast<int64_t>(row) * a.biases;
  auto shape = [&](float x, uint32_t c, int at) {
    if (c == 0) return x;
    const uint32_t made = c & ~(kSeen | kBiased);
    if (a.repetition && (c & ~kBiased)) x = x > 0.0f ? x / repetition : x * repetition;
    if (made && a.frequency) x -= frequency * static_cast<float>(made);
    if (made && a.presence) x -= presence;
    if (c & kBiased) x += bias_values[bias_at[at]];
    return x;
  };
  auto one = [&](T x, uint32_t bit, int i) {
    out[i] = from_float<T>(bit & 1u ? shape(to_float(x), counted ? counts[i] : 0u, i) : kNegInf);
  };
  if (has_edge) one(edge_value, edge_bits, edge);
  if (kVec == 1) {
    for (int i = tid + kThreads; i < size; i += kThreads) one(in[i], bits(i, false), i);
    return;
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int i = (tid + s * kThreads) * kVec;
    if (i >= rest) break;
    if (kShifted && i < whole) continue;
    const uint32_t word = words[s];
    uint32_t c[kVec];
#pragma unroll
    for (int e = 0; e < kVec; e += 4) {
      const uint4 q = counted ? *reinterpret_cast<const uint4*>(counts + i + e) : uint4{0u, 0u, 0u, 0u};
      c[e] = q.x;
      c[e + 1] = q.y;
      c[e + 2] = q.z;
      c[e + 3] = q.w;
    }
    Vec<T, kVec> x = held[s];
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      x.v[e] = word >> e & 1u ? from_float<T>(shape(to_float(x.v[e]), c[e], i + e)) : from_float<T>(kNegInf);
    *reinterpret_cast<Vec<T, kVec>*>(out + i) = x;
  }
}

// How rows lie in vectors of 16 bytes; kSingle: taken value by value.
enum class Rows { kAligned, kShifted, kSingle };

template <typename T, typename Token>
int32_t launch(const LogitsArgs& a, int batch, Rows rows, void* stream) {
  constexpr int kWide = 16 / sizeof(T);
  const int most = a.vocab + (rows == Rows::kShifted ? kWide - 1 : 0);
  const dim3 grid(batch, (most + a.tile - 1) / a.tile);
  const size_t lds = sizeof(uint32_t) * a.tile * (a.biases ? 2 : a.history ? 1 : 0);
  switch (rows) {
    case Rows::kAligned:
      hipLaunchKernelGGL((shape_logits_kernel<T, Token, kWide, false>), grid, dim3(kThreads), lds, as_stream(stream), a);
      break;
    case Rows::kShifted:
      hipLaunchKernelGGL((shape_logits_kernel<T, Token, kWide, true>), grid, dim3(kThreads), lds, as_stream(stream), a);
      break;
    default:
      hipLaunchKernelGGL((shape_logits_kernel<T, Token, 1, false>), grid, dim3(kThreads), lds, as_stream(stream), a);
  }
  return check_launch("shape_logits");
}

template <typename T>
int32_t dispatch(const LogitsArgs& a, int batch, int token_bytes, Rows rows, void* stream) {
  return token_bytes == 8 ? launch<T, int64_t>(a, batch, rows, stream)
                          : launch<T, int32_t>(a, batch, rows, stream);
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
  if (vocab > 1 << 28) return fail(PG_ERROR_UNSUPPORTED, "at most 2^28 tokens of vocabulary");
  if (dtype < PG_DTYPE_FP16 || dtype > PG_DTYPE_FP32)
    return fail(PG_ERROR_INVALID_ARGUMENT, "logits must be FP16, BF16 or FP32");
  if (history && (!history_lengths || history_capacity < 0))
    return fail(PG_ERROR_INVALID_ARGUMENT, "a history needs its lengths");
  if (history_capacity >= 1 << 30) return fail(PG_ERROR_UNSUPPORTED, "histories must be shorter than 2^30 tokens");
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
  // tiles of 8192 tokens, which read the history least often, down to 1024 where
  // 256 CUs would not get one each (histories of 4096: 8 rows of 131072 4.5 us, with
  // tiles of 8192 5.3; 4 of 32768 3.8 and 4.9; but 16 of 131072 6.4 with 4096, 6.0)
  a.tile = kMaxTile;
  while (a.tile > kMinTile && static_cast<int64_t>(batch) * ((vocab + a.tile - 1) / a.tile) < 256) a.tile /= 2;
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
  const uintptr_t first = reinterpret_cast<uintptr_t>(logits), out_first = reinterpret_cast<uintptr_t>(out);
  const bool strided = batch > 1;
  // tiles of a value per thread need no vectors, whose threads would be few (4 rows of
  // 32768 4.1 us, with vectors 4.7)
  Rows rows = Rows::kSingle;
  if (a.tile > kThreads) {
    if (first % 16 == 0 && out_first % 16 == 0 &&
        !(strided && (logits_stride * size % 16 || out_stride * size % 16)))
      rows = Rows::kAligned;
    else if ((first - out_first) % 16 == 0 && !(strided && (logits_stride - out_stride) * size % 16))
      rows = Rows::kShifted;
  }
  switch (dtype) {
    case PG_DTYPE_FP16: return dispatch<__half>(a, batch, token_bytes, rows, stream);
    case PG_DTYPE_BF16: return dispatch<__hip_bfloat16>(a, batch, token_bytes, rows, stream);
    default: return dispatch<float>(a, batch, token_bytes, rows, stream);
  }
}
