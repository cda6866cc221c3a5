// Rotary positions of query and key rows: pairs (i, i + R/2) or (2i, 2i + 1)
// of the first R dims of a head, turned by position * f_i, the remaining dims
// copied.
//
//   a' = A (a cos - b sin),  b' = A (b cos + a sin)
//
// in float32 with one rounding to the rows' type; A is the amplitude of a
// context stretched in parts.  The angles come from float64 frequencies (no
// table of positions is read or kept), and a thread turns the same kVec pairs
// of several heads of one token, so their sines are worked out once for them.
//
// Bound by HBM, and for few tokens by one trip to it.  16384 tokens of 32 query
// and 8 KV heads in FP16 (336 MB) take 70 to 72 us, 4.7 TB/s, where a copy of as
// many bytes takes 65; 8 tokens 3.7 us.  Measured and not taken at that size:
// one slice of all heads 75.5 us, 8 and 20 slices 72.8 and 79.7 (the sines over
// again), nontemporal stores 72.9, 2 or 10 heads in flight for 4 the same.
#include "pg_rotary.h"

#include <hip/hip_bf16.h>

#include <algorithm>

namespace pg {
namespace {

constexpr int kThreads = 256;

struct RotaryRows {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;   // strides in elements
  int heads;
};

struct RotaryArgs {
  RotaryRows rows[2];          // query, key (heads 0: none)
  const void* positions;       // int32 or int64 [tokens]
  const double* turns;         // revolutions per position, [rotary_dim / 2]
  float amplitude;
  int64_t tokens;
  int rotary_dim;
  int units;                   // of 2 * kVec dims of a head: pairs to turn, then dims to copy
  int turned_units;
  int heads_per_slice;         // of query and key heads together, by blockIdx.y
  int wide_positions;
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

template <typename T, int kVec, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotaryArgs a) {
  using V = Vec<T, kVec>;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t token = index / a.units;
  if (token >= a.tokens) return;
  const int unit = static_cast<int>(index - token * a.units);
  const bool turned = unit < a.turned_units;
  // the two vectors of a unit: the halves' pairs apart, everything else adjacent
  const int first = kInterleaved || !turned ? 2 * kVec * unit : kVec * unit;
  const int second = kInterleaved || !turned ? first + kVec : first + a.rotary_dim / 2;
  float2 cs[kVec];
  if (turned) {
    const int64_t position = a.wide_positions ? static_cast<const int64_t*>(a.positions)[token]
                                              : static_cast<const int32_t*>(a.positions)[token];
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      cs[i] = rotary_cos_sin(position, a.turns[unit * kVec + i], a.amplitude);
  }
  const int begin = blockIdx.y * a.heads_per_slice;
  const int end = min(begin + a.heads_per_slice, a.rows[0].heads + a.rows[1].heads);
#pragma unroll 4
  for (int h = begin; h < end; ++h) {
    const bool is_key = h >= a.rows[0].heads;
    const RotaryRows& r = a.rows[is_key];
    const int head = is_key ? h - a.rows[0].heads : h;
    const T* in = static_cast<const T*>(r.in) + token * r.in_token + head * r.in_head;
    T* out = static_cast<T*>(r.out) + token * r.out_token + head * r.out_head;
    const V x = *reinterpret_cast<const V*>(in + first);
    const V y = *reinterpret_cast<const V*>(in + second);
    V u = x, w = y;
    if (turned) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        // pair i of the unit: (x_i, y_i), or interleaved elements 2i, 2i + 1 of x, y
        const int p = 2 * i, q = 2 * i + 1;
        const T pa = !kInterleaved ? x.v[i] : p < kVec ? x.v[p % kVec] : y.v[p % kVec];
        const T pb = !kInterleaved ? y.v[i] : q < kVec ? x.v[q % kVec] : y.v[q % kVec];
        const float2 turned_pair = rotate_pair(to_float(pa), to_float(pb), cs[i]);
        const T ra = from_float<T>(turned_pair.x);
        const T rb = from_float<T>(turned_pair.y);
        if (!kInterleaved) {
          u.v[i] = ra;
          w.v[i] = rb;
        } else {
          (p < kVec ? u.v[p % kVec] : w.v[p % kVec]) = ra;
          (q < kVec ? u.v[q % kVec] : w.v[q % kVec]) = rb;
        }
      }
    }
    *reinterpret_cast<V*>(out + first) = u;
    *reinterpret_cast<V*>(out + second) = w;
  }
}

template <typename T, int kVec>
void launch(const RotaryArgs& a, bool interleaved, const dim3& grid, void* stream) {
  if (interleaved)
    hipLaunchKernelGGL((rotate_kernel<T, kVec, true>), grid, dim3(kThreads), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL((rotate_kernel<T, kVec, false>), grid, dim3(kThreads), 0, as_stream(stream), a);
}

template <typename T>
int32_t dispatch(RotaryArgs a, int vec, int head_dim, bool interleaved, void* stream) {
  a.turned_units = a.rotary_dim / 2 / vec;
  const bool copies = a.rows[0].in != a.rows[0].out || (a.rows[1].heads && a.rows[1].in != a.rows[1].out);
  a.units = a.turned_units + (copies ? (head_dim - a.rotary_dim) / (2 * vec) : 0);
  const int64_t blocks = (a.tokens * a.units + kThreads - 1) / kThreads;
  if (blocks > UINT32_MAX / kThreads) return fail(PG_ERROR_UNSUPPORTED, "too many rows for one rotation");
  const int heads = a.rows[0].heads + a.rows[1].heads;
  // few tokens: the heads of a token over several workgroups, up to 2048 in all (40
  // heads of 8 tokens 2.8 us, in one slice 17.5; of 1024 6.6 and 20.1)
  int slices = static_cast<int>(std::min<int64_t>(heads, std::max<int64_t>(1, 2048 / blocks)));
  a.heads_per_slice = (heads + slices - 1) / slices;
  slices = (heads + a.heads_per_slice - 1) / a.heads_per_slice;
  const dim3 grid(static_cast<uint32_t>(blocks), slices);
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2) launch<T, 8>(a, interleaved, grid, stream);
      break;
    case 4: launch<T, 4>(a, interleaved, grid, stream); break;
    case 2: launch<T, 2>(a, interleaved, grid, stream); break;
    default: launch<T, 1>(a, interleaved, grid, stream); break;
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
  if (query_heads > 65535 || key_heads > 65535 || head_dim > 65536)
    return fail(PG_ERROR_UNSUPPORTED, "at most 65535 heads of 65536 dims");
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
