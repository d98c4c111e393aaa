// Element formats of the paged KV cache: conversions between the stored one-byte rows and MMA operands.
#pragma once
#include "common.cuh"

namespace q35 {

__device__ __forceinline__ uint32_t cvt_e4m3x2_f16x2(uint32_t two_bytes) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((unsigned short)two_bytes));
  return d;
}

// two one-byte FP8 cache elements (bytes I0, I1 of x) as f16x2
template <int I0, int I1>
__device__ __forceinline__ uint32_t cvt_kv(uint32_t x) {
  return cvt_e4m3x2_f16x2(__byte_perm(x, 0, 0x4400 | I0 | (I1 << 4)));
}

// int8 bytes I0, I1 of xs (= x ^ 0x80808080) times their rows' scales, rounded to bf16 -- bf16(int8 * scale), the
// reference's page dequantisation (kv_page, models/qwen38_27b/decode/q35_group.py:208-222), exactly: 0x4B000000 | b is
// the float 2^23 + b, the fused multiply-add against -(2^23 + 128) * s leaves (b - 128) * s, a 15-bit product that
// fp32 holds exactly, and one cvt.rn rounds the pair.
template <int I0, int I1>
__device__ __forceinline__ uint32_t cvt_s8x2_bf16x2(uint32_t xs, float s0, float s1) {
  const float f0 = __uint_as_float(__byte_perm(xs, 0x4B000000u, 0x7540 | I0));
  const float f1 = __uint_as_float(__byte_perm(xs, 0x4B000000u, 0x7540 | I1));
  return pack_bf16(fmaf(f0, s0, -8388736.f * s0), fmaf(f1, s1, -8388736.f * s1));
}

}  // namespace q35
