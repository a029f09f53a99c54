// MXFP4 blocks (OCP Microscaling Formats 1.0): 32 e2m1 elements under one e8m0
// scale, quantised in registers. Shared by the codec and the product of two
// MXFP4 operands.
#pragma once

#include "common.h"

namespace mx {
namespace mxfp4 {

constexpr int kBlock = 32;

// The maximum over the 4 lanes of a quad, in all of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xf, 0xf, true)));
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xf, 0xf, true)));
}

// Eight elements of a block whose four groups of 8 sit in the lanes of a quad:
// their codes (element 0 in the low nibble) and the block's scale byte. The
// maximum is taken over the bits of |x|, so that a NaN, whose bits are the largest,
// is kept. floor(log2 max) is the exponent field, and the scale byte that field
// less 2 (0 for denormals and zero: 2^-127).
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], uint32_t &scale) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
  const uint32_t field = quad_max(a) >> 23;
  scale = field == 255 ? 255 : field > 2 ? field - 2 : 0;
  if (field == 255) return 0;
  // 2^-127 is a denormal.
  const float s = __uint_as_float(scale == 0 ? 0x00400000u : scale << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
  return c;
}

// Eight elements from p on as fp32.
template <bool BF16>
__device__ __forceinline__ void load8(const void *p, int64_t at, float (&v)[8]) {
  if constexpr (BF16) {
    const u32x4 q = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
    }
  } else {
    const f32x4_any *q = reinterpret_cast<const f32x4_any *>(static_cast<const float *>(p) + at);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[i + 4] = b[i];
    }
  }
}

// The first n <= 8 of eight elements, the others zero.
template <bool BF16>
__device__ __forceinline__ void load8_guarded(const void *p, int64_t at, int n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (BF16)
      v[i] = i < n ? bf16_bits_to_f32(static_cast<const uint16_t *>(p)[at + i]) : 0.0f;
    else
      v[i] = i < n ? static_cast<const float *>(p)[at + i] : 0.0f;
  }
}

}  // namespace mxfp4
}  // namespace mx
