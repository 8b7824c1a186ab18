// The 8-bit paged KV cache: formats, tile order and conversions.
//
// A cached row (one token, one kv head, K or V, D bf16 numbers x with largest magnitude a) is D codes and one fp32 scale:
//   KV_INT8  code = rne(127 x / a)         scale = a / 127
//   KV_FP8   code = e4m3(448 x / a), rne   scale = a / 448
// A row of zeros has scale 0; a row that holds an infinity or NaN has scale NaN and codes 0, so it reads back as NaN throughout.
//
// codes [num_blocks, Hkv, block_size, D] bytes, K and V; scales [num_blocks, Hkv, 2, block_size] fp32 (K's, then V's: both of a
// 16-token page share one 128-byte line). The D x 16 codes of 16 tokens ("tile", token t of 0..15) lie in the order in which the
// matrix instructions take them, so an attention kernel loads a tile with whole 1 KiB wave reads and feeds it without LDS:
//   K  byte (t, d) at ((d / 16) 16 + t) 16 + d % 16
//      lane (g, li) reads 16 bytes: token li, dims 16 (4 i + g) .. + 16, of load i: two A fragments of S^T = K Q^T
//   V  byte (t, d) at ((d / 64) 64 + 16 (t / 4) + d % 16) 16 + (d / 16) % 4 * 4 + t % 4
//      lane (g, li) reads tokens 4 g .. + 4 of dims 64 i + {0, 16, 32, 48} + li: A fragments of O^T = V^T P^T
#pragma once

#include "common.h"

namespace xgk {

enum : int { KV_BF16 = 0, KV_FP8 = 1, KV_INT8 = 2 };

constexpr int KV_TILE = 16;

__device__ __forceinline__ int kv_k_byte(int t, int d) { return ((d >> 4) * 16 + t) * 16 + (d & 15); }
__device__ __forceinline__ int kv_v_byte(int t, int d) {
  return ((d >> 6) * 64 + 16 * (t >> 2) + (d & 15)) * 16 + ((d >> 4) & 3) * 4 + (t & 3);
}

// four codes -> four bf16 (exact: E4M3 values and integers up to 127 are bf16 numbers)
template <int FMT>
__device__ __forceinline__ uint2 kv_widen4(uint32_t w) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (FMT == KV_FP8) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
  } else {
    const float a = static_cast<float>(static_cast<int8_t>(w & 0xFF));
    const float b = static_cast<float>(static_cast<int8_t>((w >> 8) & 0xFF));
    const float c = static_cast<float>(static_cast<int8_t>((w >> 16) & 0xFF));
    const float d = static_cast<float>(static_cast<int8_t>(w >> 24));
    // (whole numbers: the bf16 of each is its upper half)
    return make_uint2(__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u),
                      __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x07060302u));
  }
#else
  return make_uint2(0, 0);
#endif
}

template <int FMT>
__device__ __forceinline__ bf16x8_t kv_widen8(uint32_t lo, uint32_t hi) {
  const uint2 a = kv_widen4<FMT>(lo), b = kv_widen4<FMT>(hi);
  return as_frag(make_uint4(a.x, a.y, b.x, b.y));
}

}  // namespace xgk
