// Arithmetic shared by the quant kernels (per-token rows and 128-value blocks): the scale's bounds and division, bf16
// unpacking, and packed abs-max and e4m3 conversion of 8 bf16 values.
#pragma once

#include "common.cuh"

namespace h3b {

static constexpr float kFp8Max = 448.0f;
static constexpr float kMinScale = 1.0f / (448.0f * 512.0f);

__device__ __forceinline__ float qdiv(float a, float b, int mode) {
  return mode == H3B_DIV_FULL ? div_full(a, b) : __fdiv_rn(a, b);
}

__device__ __forceinline__ float lo_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// running abs-max of 8 bf16 values, kept as two packed 16-bit unsigned maxima
__device__ __forceinline__ uint32_t absmax8(const uint4& v, uint32_t m2) {
  m2 = __vmaxu2(m2, v.x & 0x7FFF7FFFu);
  m2 = __vmaxu2(m2, v.y & 0x7FFF7FFFu);
  m2 = __vmaxu2(m2, v.z & 0x7FFF7FFFu);
  m2 = __vmaxu2(m2, v.w & 0x7FFF7FFFu);
  return m2;
}
__device__ __forceinline__ uint32_t fold16(uint32_t m2) { return max(m2 & 0xFFFFu, m2 >> 16); }

// 8 bf16 -> 8 e4m3 (one 8-byte word): x * inv, round to nearest even; satfinite clamps to +-448 exactly as the
// reference's clamp does for every finite or infinite product, and keeps NaN
__device__ __forceinline__ uint2 quant8(const uint4& v, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t a = f32x2_to_e4m3x2(lo_bf16(w[2 * i]) * inv, hi_bf16(w[2 * i]) * inv);
    const uint16_t b = f32x2_to_e4m3x2(lo_bf16(w[2 * i + 1]) * inv, hi_bf16(w[2 * i + 1]) * inv);
    o[i] = static_cast<uint32_t>(a) | (static_cast<uint32_t>(b) << 16);
  }
  return make_uint2(o[0], o[1]);
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo_bf16(w[i]);
    f[2 * i + 1] = hi_bf16(w[i]);
  }
}

}  // namespace h3b
