// Rotary positions of query and key rows: pairs (i, i + R/2) or (2i, 2i + 1)
// of the first R dims of a head, turned by position * f_i, the remaining dims
// copied.
//
//   a' = A (a cos - b sin),  b' = A (b cos + a sin)
//
// in float32 with one rounding to the rows' type; A is the amplitude of a
// context stretched in parts.  The angles come from float64 frequencies: no
// table of positions is read or kept.
//
// Bound by HBM, and for few tokens by one trip to it.  16384 tokens of 32 query
// and 8 KV heads in FP16 (336 MB) take 63.6 us, 5.3 TB/s, where a copy of as many
// bytes takes 62.8; 8 tokens 2.9 us (with the gap between launches).  What it takes
// is many short workgroups that walk through memory in order: threads that keep
// their pairs and stride over the heads of a token took 70.9 us, workgroups of 640
// units with 2 or 4 in flight per thread 65.9 and 69, and longer ones (1280, 2560)
// 64.3 and 69.
#include "pg_rotary.h"
#include "pg_types.h"

#include <algorithm>

namespace pg {
namespace {

constexpr int kThreads = 256;
constexpr int kBlockUnits = 640;          // of a workgroup, where there are many
constexpr int kMaxPairs = 4096;           // of tokens that share a workgroup, 32 KiB of LDS
constexpr int kMaxUnits = 60000;          // of a workgroup
// A token by itself may have more pairs; its sines fill at most the LDS that a launch
// gets without asking for more, and its head is one slice.
constexpr int kMaxHeadDim = 16384;
static_assert(sizeof(float2) * (kMaxHeadDim / 2) <= 64 * 1024 && kMaxPairs <= kMaxHeadDim / 2, "LDS of a workgroup");
static_assert(kMaxHeadDim / 2 <= kMaxUnits, "units of a head");
constexpr int64_t kFull = 2048 * kThreads;     // units of a call

struct RotaryRows {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;   // strides in elements
  int heads;
};

// Quotients of small numbers: n / d = mulhi(n, 2^32 / d rounded up) while n * d
// stays below 2^32.
struct Divisor {
  uint32_t d, m;
  static Divisor by(uint32_t d) { return {d, d > 1 ? static_cast<uint32_t>((0x100000000ull + d - 1) / d) : 0}; }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return d > 1 ? __umulhi(n, m) : n; }
};

struct RotaryArgs {
  RotaryRows rows[2];          // query, key (heads 0: none)
  const void* positions;       // int32 or int64 [tokens]
  const double* turns;         // revolutions per position, [rotary_dim / 2]
  float amplitude;
  int64_t tokens;
  int rotary_dim;
  int turned_units;            // units of 2 * kVec dims of a head: pairs to turn, then dims to copy
  int heads_per_slice;         // of query and key heads together, by blockIdx.y
  int tokens_per_block;
  int wide_positions;
  Divisor pairs, units, slice; // rotary_dim / 2, units of a head, heads_per_slice
};

// A workgroup takes the heads of a slice of a few tokens: their sines once, into
// LDS, while the first rows are on their way, then unit by unit in the order of
// memory (a unit is 2 * kVec dims).
template <typename T, int kVec, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotaryArgs a) {
  using V = Vec<T, kVec>;
  extern __shared__ __attribute__((aligned(16))) float2 cos_sin[];   // [tokens][pairs]
  const int64_t first_token = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_block), a.tokens - first_token));
  const int first_head = blockIdx.y * a.heads_per_slice;
  const int heads = min(a.heads_per_slice, a.rows[0].heads + a.rows[1].heads - first_head);
  const uint32_t tid = threadIdx.x;
  const uint32_t total = static_cast<uint32_t>(tokens * a.heads_per_slice) * a.units.d;

  struct Place {
    int token, unit, first, second;    // first, second: dims of the unit's two vectors
    bool turned, is_key, valid;
    int head;
  };
  // unit ``n`` of the workgroup; of a slice short of heads some are missing
  auto place = [&](uint32_t n) {
    Place p;
    const uint32_t row = a.units.of(n);
    p.unit = n - row * a.units.d;
    p.token = a.slice.of(row);
    const int h = row - p.token * a.slice.d;
    p.valid = n < total && h < heads;
    const int head = first_head + (p.valid ? h : 0);
    p.token = n < total ? p.token : 0;
    p.is_key = head >= a.rows[0].heads;
    p.head = p.is_key ? head - a.rows[0].heads : head;
    p.turned = p.unit < a.turned_units;
    // the halves' pairs lie apart, everything else side by side
    p.first = kInterleaved || !p.turned ? 2 * kVec * p.unit : kVec * p.unit;
    p.second = kInterleaved || !p.turned ? p.first + kVec : p.first + a.rotary_dim / 2;
    return p;
  };
  V x, y;
  auto request = [&](const Place& p) {
    const RotaryRows& r = a.rows[p.is_key];
    const T* in = static_cast<const T*>(r.in) + (first_token + p.token) * r.in_token + p.head * r.in_head;
    x = *reinterpret_cast<const V*>(in + p.first);
    y = *reinterpret_cast<const V*>(in + p.second);
  };
  Place p = place(tid);
  request(p);
  for (uint32_t i = tid; i < tokens * a.pairs.d; i += kThreads) {
    const uint32_t token = a.pairs.of(i);
    const int64_t position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[first_token + token]
                                              : static_cast<const int32_t*>(a.positions)[first_token + token];
    cos_sin[i] = rotary_cos_sin(position, a.turns[i - token * a.pairs.d], a.amplitude);
  }
  __syncthreads();
  for (uint32_t n = tid;;) {
    if (p.valid) {
      V u = x, w = y;
      if (p.turned) {
        const float2* cs = cos_sin + p.token * a.pairs.d + p.unit * kVec;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          // pair i of the unit: (x_i, y_i), or interleaved elements 2i, 2i + 1 of x, y
          const int e = 2 * i, o = 2 * i + 1;
          const T pa = !kInterleaved ? x.v[i] : e < kVec ? x.v[e % kVec] : y.v[e % kVec];
          const T pb = !kInterleaved ? y.v[i] : o < kVec ? x.v[o % kVec] : y.v[o % kVec];
          const float2 turned_pair = rotate_pair(to_float(pa), to_float(pb), cs[i]);
          const T ra = from_float<T>(turned_pair.x);
          const T rb = from_float<T>(turned_pair.y);
          if (!kInterleaved) {
            u.v[i] = ra;
            w.v[i] = rb;
          } else {
            (e < kVec ? u.v[e % kVec] : w.v[e % kVec]) = ra;
            (o < kVec ? u.v[o % kVec] : w.v[o % kVec]) = rb;
          }
        }
      }
      const RotaryRows& r = a.rows[p.is_key];
      T* out = static_cast<T*>(r.out) + (first_token + p.token) * r.out_token + p.head * r.out_head;
      *reinterpret_cast<V*>(out + p.first) = u;
      *reinterpret_cast<V*>(out + p.second) = w;
    }
    n += kThreads;
    if (n >= total) return;
    p = place(n);
    request(p);
  }
}

template <typename T, int kVec>
void launch(const RotaryArgs& a, bool interleaved, const dim3& grid, size_t lds, void* stream) {
  if (interleaved)
    hipLaunchKernelGGL((rotate_kernel<T, kVec, true>), grid, dim3(kThreads), lds, as_stream(stream), a);
  else
    hipLaunchKernelGGL((rotate_kernel<T, kVec, false>), grid, dim3(kThreads), lds, as_stream(stream), a);
}

template <typename T>
int32_t dispatch(RotaryArgs a, int vec, int head_dim, bool interleaved, void* stream) {
  a.turned_units = a.rotary_dim / 2 / vec;
  const bool copies = a.rows[0].in != a.rows[0].out || (a.rows[1].heads && a.rows[1].in != a.rows[1].out);
  const int units = a.turned_units + (copies ? (head_dim - a.rotary_dim) / (2 * vec) : 0);
  const int heads = a.rows[0].heads + a.rows[1].heads;
  const int64_t per_token = static_cast<int64_t>(heads) * units;
  // Whole tokens of 640 units per workgroup, where there are many, and of one per
  // thread otherwise; a token of more than that is cut at its heads (8 tokens of 40
  // heads 2.9 us, whole 3.4; 1024 5.6 and 6.2; but 4096 16.4 and 15.0).
  const bool many = a.tokens * per_token >= kFull;
  const int64_t fit = (many ? kBlockUnits : kThreads) / per_token;
  a.tokens_per_block = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(fit, kMaxPairs / (a.rotary_dim / 2))));
  a.heads_per_slice = many ? heads : std::min(heads, std::max(1, kThreads / units));
  // numbers and divisors of place() stay below 2^16
  a.heads_per_slice = std::min(a.heads_per_slice, std::max(1, kMaxUnits / units));
  a.pairs = Divisor::by(a.rotary_dim / 2);
  a.units = Divisor::by(units);
  a.slice = Divisor::by(a.heads_per_slice);
  const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (blocks > UINT32_MAX / kThreads) return fail(PG_ERROR_UNSUPPORTED, "too many rows for one rotation");
  const dim3 grid(static_cast<uint32_t>(blocks), (heads + a.heads_per_slice - 1) / a.heads_per_slice);
  const size_t lds = sizeof(float2) * a.tokens_per_block * (a.rotary_dim / 2);
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) launch<T, 8>(a, interleaved, grid, lds, stream);
      break;
    case 4: launch<T, 4>(a, interleaved, grid, lds, stream); break;
    case 2: launch<T, 2>(a, interleaved, grid, lds, stream); break;
    default: launch<T, 1>(a, interleaved, grid, lds, stream); break;
  }
  return check_launch("rotate");
}

}  // namespace
}  // namespace pg

using namespace pg;

extern "C" int32_t pg_rotate(const void* query, int64_t query_token_stride,
                             int64_t query_head_stride, int32_t query_heads, const void* key,
                             int64_t key_token_stride, int64_t key_head_stride, int32_t key_heads,
                             void* out_query, int64_t out_query_token_stride,
                             int64_t out_query_head_stride, void* out_key,
                             int64_t out_key_token_stride, int64_t out_key_head_stride,
                             const void* positions, int32_t position_bytes, const double* turns,
                             float amplitude, int64_t tokens, int32_t head_dim, int32_t rotary_dim,
                             int32_t interleaved, int32_t dtype, void* stream) {
  clear_error();
  if (query_heads < 0 || key_heads < 0 || tokens < 0 || query_heads + static_cast<int64_t>(key_heads) <= 0)
    return fail(PG_ERROR_INVALID_ARGUMENT, "token and head counts must be nonnegative, with a head");
  if (query_heads > 65535 || key_heads > 65535 || head_dim > kMaxHeadDim)
    return fail(PG_ERROR_UNSUPPORTED, "at most 65535 heads of 16384 dims");
  if (!positions || !turns || (query_heads && (!query || !out_query)) || (key_heads && (!key || !out_key)))
    return fail(PG_ERROR_INVALID_ARGUMENT, "null tensor pointer");
  if (rotary_dim <= 0 || rotary_dim % 2 || head_dim % 2 || rotary_dim > head_dim)
    return fail(PG_ERROR_INVALID_ARGUMENT, "the rotated part must be an even number of a head's dims");
  if (position_bytes != 4 && position_bytes != 8)
    return fail(PG_ERROR_INVALID_ARGUMENT, "positions must be int32 or int64");
  if (dtype < PG_DTYPE_FP16 || dtype > PG_DTYPE_FP32)
    return fail(PG_ERROR_INVALID_ARGUMENT, "rows must be FP16, BF16 or FP32");
  if (tokens == 0) return PG_OK;
  RotaryArgs a{};
  a.rows[0] = {query, out_query, query_token_stride, query_head_stride, out_query_token_stride,
               out_query_head_stride, query_heads};
  a.rows[1] = {key, out_key, key_token_stride, key_head_stride, out_key_token_stride,
               out_key_head_stride, key_heads};
  a.positions = positions;
  a.turns = turns;
  a.amplitude = amplitude;
  a.tokens = tokens;
  a.rotary_dim = rotary_dim;
  a.wide_positions = position_bytes == 8;
  // the widest vectors, up to 16 bytes, that the pairs, the copied dims and
  // every row's alignment allow
  const int size = dtype == PG_DTYPE_FP32 ? 4 : 2;
  int vec = 16 / size;
  auto fits = [&](int v) {
    if (rotary_dim / 2 % v || (head_dim - rotary_dim) % (2 * v)) return false;
    for (const RotaryRows& r : a.rows) {
      if (!r.heads) continue;
      if (r.in_token % v || r.in_head % v || r.out_token % v || r.out_head % v) return false;
      if (reinterpret_cast<uintptr_t>(r.in) % (v * size) || reinterpret_cast<uintptr_t>(r.out) % (v * size))
        return false;
    }
    return true;
  };
  while (vec > 1 && !fits(vec)) vec /= 2;
  switch (dtype) {
    case PG_DTYPE_FP16: return dispatch<__half>(a, vec, head_dim, interleaved != 0, stream);
    case PG_DTYPE_BF16: return dispatch<__hip_bfloat16>(a, vec, head_dim, interleaved != 0, stream);
    default: return dispatch<float>(a, vec, head_dim, interleaved != 0, stream);
  }
}
