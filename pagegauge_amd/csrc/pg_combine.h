// The second half of a split attention: partial softmax states of a request's work
// items joined, the value center added.
#pragma once

#include "pg_common.h"

namespace pg {
namespace {

constexpr float kNoScore = -__builtin_huge_valf();

struct CombineArgs {
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
  int written;                     // requests of so many items were written by their workgroups
};

// Joins the partial states of one (request, query head), 64 dims a workgroup:
// thread (row, column) = (tid / 16, tid % 16) takes items row, row + 16, ... of
// four dims.  The first 64 items are requested together, so a join of that many
// is one trip to memory after the item range.
constexpr int kCombineThreads = 256;
constexpr int kCombineRows = kCombineThreads / 16;
constexpr int kCombineInFlight = 4;

__global__ __launch_bounds__(kCombineThreads) void combine_kernel(CombineArgs a) {
  constexpr int kWaves = kCombineThreads / kWave;
  __shared__ float part_o[kWaves][64];
  __shared__ float part_m[kWaves], part_l[kWaves];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int row = threadIdx.x / 16, dim = 64 * blockIdx.z + 4 * (threadIdx.x % 16);
  const int request = blockIdx.x, head = blockIdx.y;
  const int begin = a.single ? 0 : a.item_ptr[request];
  const int end = a.single ? a.single : a.item_ptr[request + 1];
  if (end - begin <= a.written) return;
  float m = kNoScore, l = 0.0f;
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
      if (first + k * kCombineRows >= end) mi[k] = kNoScore;
      top = fmaxf(top, mi[k]);
    }
    const float base = top == kNoScore ? 0.0f : top;
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
  const float base = top == kNoScore ? 0.0f : top;
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
  float all = kNoScore;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all = fmaxf(all, part_m[w]);
  const float all_base = all == kNoScore ? 0.0f : all;
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
  if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? kNoScore : log2f(sum) + all;
}

}  // namespace
}  // namespace pg
