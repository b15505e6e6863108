// Arithmetic shared by the quant kernels (per-token rows and 128-value blocks): the scale's bounds and division, bf16
// unpacking, and the fold of a packed abs-max.
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

__device__ __forceinline__ uint32_t fold16(uint32_t m2) { return max(m2 & 0xFFFFu, m2 >> 16); }

}  // namespace h3b
