// The cache held in 4 bits: its layout, shared by the kernels that write it
// (pg_int4_cache.hip) and the attention that reads it (pg_int4_decode.hip).
//
// One (page, KV head) block holds 16 tokens x 128 dims of K, then of V, 1024
// bytes each, and 64 bytes of scales elsewhere:
//   codes   uint8 [pages, Hkv, 2 (K, V), 1024]
//   scales  FP16  [pages, Hkv, 4 (token group kg), 2 (K, V), 4]
// A token's 128 values of a head share one scale, and a nibble holds code + 8
// with code in [-7, 7].
//
// Pages are written whole (from the exact FP16 page that a token completed, or
// from a prompt) and so need no token-major rows: each block lies in the order
// in which a wave's lanes feed it to v_mfma_f32_16x16x32_f16.  Lane (kg, n) =
// (lane / 16, lane % 16) owns 16 bytes at 16 * lane of the K and of the V part,
// so that each is one 1 KiB load of the wave:
//   K: token n, dims 32 w + 8 kg + e of dword w, e = 0..7
//   V: tokens 4 kg + t, t = 0..3, of channels 8 n + 2 j and 8 n + 2 j + 1 of dword j
// Within a dword, shifting by 4 i and masking with 0x000f000f leaves one pair of
// MFMA neighbours in the two halves:
//   K: nibble i     = dim 2 i, nibble i + 4 = dim 2 i + 1           (e = 2 i, 2 i + 1)
//   V: nibbles 0, 4 = tokens 0, 1 and 1, 5 = tokens 2, 3 of channel 8 n + 2 j;
//      nibbles 2, 6 and 3, 7 likewise of channel 8 n + 2 j + 1
#pragma once

#include "pg_common.h"

namespace pg {

constexpr int kInt4PartBytes = 1024;                  // K or V of a (page, head) block
constexpr int kInt4BlockBytes = 2 * kInt4PartBytes;
constexpr int kInt4BlockScales = 32;                  // FP16 scales of a block

// Element of a block's scales: token ``t`` of K (part 0) or V (part 1).
__host__ __device__ constexpr int int4_scale_index(int part, int t) {
  return (t >> 2) * 8 + part * 4 + (t & 3);
}

}  // namespace pg
