// Block-scaled FP8 quantisation (HBM bound): e4m3 values with one fp32 scale for each 128 consecutive values of a row
// (activations; plain, or of silu(gate) * up) or for each 128 x 128 tile (weights).  The scale and the rounding are
// those of the per-token quant, taken over a block:
//   scale = max(amax / 448, 1/(448*512)),  q = e4m3_rn(clamp(h * (1 / scale), -448, 448))     (NaN propagates)
//
// Activations: 16 lanes hold a block as one 16-byte load each (8 bf16 values), reduce its abs-max inside the half-warp and
// write 128 bytes of e4m3; no shared memory, no barrier.  A warp takes the same block of eight consecutive rows: blocks
// taken along a row instead, each with divisions and a 4-byte scale store of its own, ran at 4.9 TB/s (62,496 x 5,120:
// 199 us), this at 6.4 (151 us; the copy rate is 6.46).  silu-mul, 31,248 x
// 13,824: 361 us, 6.0 TB/s (blocks along a row 466; two rows 429; CTAs of 256 threads 385).  Weights: a CTA of 256 threads
// holds a 128 x 128 tile in registers (8 vectors per thread) and reduces it once: 15,360 x 5,120 in 36 us, 6.5 TB/s (512
// threads: 50 us).  Every value is read once and written once.
#include "common.cuh"
#include "quant.cuh"

namespace h3b {
namespace {

constexpr int BLK = 128;

// 8 values of a row starting at column c, as bf16 bit patterns; VEC: one 16-byte load (K % 8 == 0, so they are all in
// the row or all past it); otherwise value by value with columns at or past K as zero
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int64_t c, int64_t K) {
  if constexpr (VEC) {
    return c < K ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = c + 2 * i < K ? row[c + 2 * i] : 0u;
      const uint32_t hi = c + 2 * i + 1 < K ? row[c + 2 * i + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(uint8_t* row, int64_t c, int64_t K, uint2 v) {
  if constexpr (VEC) {
    if (c < K) *reinterpret_cast<uint2*>(row + c) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < K) row[c + i] = static_cast<uint8_t>((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits, int div_mode) {
  return nan_max(qdiv(__uint_as_float(amax_bits), kFp8Max, div_mode), kMinScale);
}

// silu(g) * u in fp32, not rounded before the quant: one rounding, to e4m3.  The fast exponential and division are within
// (2 + 1.173 |g|) and 2 units in the last place, i.e. (6 + 1.2 |g|) * 2^-23 in all, against the 2^-4 of the rounding.
__device__ __forceinline__ float silu_mul_f32(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

__device__ __forceinline__ uint2 quant8f(const float (&y)[8], float inv) {
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint16_t a = f32x2_to_e4m3x2(y[4 * i] * inv, y[4 * i + 1] * inv);
    const uint16_t b = f32x2_to_e4m3x2(y[4 * i + 2] * inv, y[4 * i + 3] * inv);
    o[i] = static_cast<uint32_t>(a) | (static_cast<uint32_t>(b) << 16);
  }
  return make_uint2(o[0], o[1]);
}

constexpr int U = 4;  // rows of a half-warp (two: 5.5 TB/s where four make 6.4)

// Maxima of four values over the 16 lanes of a half-warp in 5 shuffles instead of 16: in each of the first two steps a lane
// gives half of its values away and keeps the other half.  Lane hl is left with the maximum of value hl / 4.
__device__ __forceinline__ uint32_t half_warp_max(const uint32_t (&v)[U], int hl) {
  static_assert(U == 4, "two halving steps");
  constexpr uint32_t ALL = 0xffffffffu;
  const bool hi = hl & 8, odd = hl & 4;
  uint32_t a = hi ? v[2] : v[0], b = hi ? v[3] : v[1];
  a = max(a, __shfl_xor_sync(ALL, hi ? v[0] : v[2], 8));
  b = max(b, __shfl_xor_sync(ALL, hi ? v[1] : v[3], 8));
  uint32_t m = max(odd ? b : a, __shfl_xor_sync(ALL, odd ? a : b, 4));
  m = max(m, __shfl_xor_sync(ALL, m, 2));
  return max(m, __shfl_xor_sync(ALL, m, 1));
}

// rows x [rows, K] (SILU: [rows, 2K], gate | up) -> q [rows, K], s[row * s_row + j * s_blk].  A warp takes block j of 2U
// consecutive rows, U per half-warp: their scales are then neighbours in the block-major scale tensor and leave in one
// store, each division is made once per warp for 2U blocks, and the loads of a CTA's 4 warps run along the rows.
template <bool VEC, bool SILU>
__global__ void __launch_bounds__(128) quant_blocks_kernel(const uint16_t* __restrict__ x, uint32_t rows, uint32_t units,
                                                           uint32_t KB, int64_t K, int64_t stride_x,
                                                           uint8_t* __restrict__ q, float* __restrict__ s, int64_t s_row,
                                                           int64_t s_blk, int div_mode) {
  pdl_wait();
  pdl_launch();
  const int hl = threadIdx.x & 15;
  const uint32_t unit = blockIdx.x * 4u + (threadIdx.x >> 5);
  if (unit >= units) return;  // the whole warp
  const uint32_t group = unit / KB, j = unit - group * KB;
  const uint32_t row0 = group * (2u * U) + (threadIdx.x & 16 ? U : 0u);
  const int64_t c = static_cast<int64_t>(j) * BLK + hl * 8;
  uint4 v[U], w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    v[u] = w[u] = make_uint4(0, 0, 0, 0);
    if (row0 + u < rows) {
      const uint16_t* xr = x + (row0 + u) * stride_x;
      v[u] = load8<VEC>(xr, c, K);
      if (SILU) w[u] = load8<VEC>(xr + K, c, K);
    }
  }
  float y[SILU ? U : 1][8];
  uint32_t amax[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if constexpr (SILU) {
      float f[8];
      unpack8(v[u], y[u]);
      unpack8(w[u], f);
      amax[u] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[u][e] = silu_mul_f32(y[u][e], f[e]);
        amax[u] = max(amax[u], __float_as_uint(y[u][e]) & 0x7FFFFFFFu);  // NaN bits sort above every number
      }
    } else {
      amax[u] = fold16(absmax8(v[u], 0)) << 16;
    }
  }
  const float scale = block_scale(half_warp_max(amax, hl), div_mode);
  const float inv = qdiv(1.0f, scale, div_mode);
  const uint32_t mine = row0 + hl / 4;
  if (hl % 4 == 0 && mine < rows) s[mine * s_row + j * s_blk] = scale;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv_u = __shfl_sync(0xffffffffu, inv, (threadIdx.x & 16) + u * 4);
    if (row0 + u < rows) {
      uint2 out;
      if constexpr (SILU)
        out = quant8f(y[u], inv_u);
      else
        out = quant8(v[u], inv_u);
      store8<VEC>(q + (row0 + u) * K, c, K, out);
    }
  }
}

// w [E, N, K] -> q [E, N, K] contiguous, s [E, NB, KB] contiguous: one CTA per tile
template <bool VEC>
__global__ void __launch_bounds__(256) quant_weight_blocks_kernel(const uint16_t* __restrict__ w, int64_t N, int64_t K,
                                                                  int64_t stride_e, int64_t stride_n, uint32_t NB,
                                                                  uint32_t KB, uint8_t* __restrict__ q,
                                                                  float* __restrict__ s, int div_mode) {
  __shared__ uint32_t red[8];
  __shared__ float tile_scale[2];  // and its inverse
  pdl_wait();
  pdl_launch();
  const uint32_t tile = blockIdx.x;
  const uint32_t j = tile % KB, en = tile / KB, i = en % NB, e = en / NB;
  const int64_t c = static_cast<int64_t>(j) * BLK + (threadIdx.x & 15) * 8;
  const int64_t r0 = static_cast<int64_t>(i) * BLK + (threadIdx.x >> 4);
  const uint16_t* we = w + e * stride_e;
  uint4 v[8];
  uint32_t m2 = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int64_t r = r0 + 16 * u;
    v[u] = r < N ? load8<VEC>(we + r * stride_n, c, K) : make_uint4(0, 0, 0, 0);
    m2 = absmax8(v[u], m2);
  }
  const uint32_t wmax = __reduce_max_sync(0xffffffffu, fold16(m2));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = wmax;
  __syncthreads();
  uint32_t amax = red[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) amax = max(amax, red[k]);
  if (threadIdx.x < 32) {  // the divisions in one warp: in all eight they took a tenth of the kernel
    const float scale = block_scale(amax << 16, div_mode);
    tile_scale[0] = scale;
    tile_scale[1] = qdiv(1.0f, scale, div_mode);
  }
  __syncthreads();
  const float inv = tile_scale[1];
  if (threadIdx.x == 0) s[tile] = tile_scale[0];  // behind the barrier: ahead of it the others waited for it, 39.4 us for 36
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int64_t r = r0 + 16 * u;
    if (r < N) store8<VEC>(q + (e * N + r) * K, c, K, quant8(v[u], inv));
  }
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int bad_mode(int div_mode) { return div_mode != H3B_DIV_IEEE && div_mode != H3B_DIV_FULL; }

template <typename... P, typename... A>
int launch(const char* what, void (*kernel)(P...), unsigned grid, unsigned threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? H3B_OK : cuda_fail(e, what);
}

template <bool SILU>
int quant_blocks(const char* what, const void* x, int64_t rows, int64_t K, int64_t stride_x, void* q, float* s,
                 int64_t s_row, int64_t s_blk, int32_t div_mode, cudaStream_t st) {
  if (rows < 0 || K < 0) return fail(H3B_EINVAL, "%s: rows %lld width %lld", what, (long long)rows, (long long)K);
  if (bad_mode(div_mode)) return fail(H3B_EINVAL, "%s: div_mode %d", what, div_mode);
  if (rows == 0 || K == 0) return H3B_OK;
  if (x == nullptr || q == nullptr || s == nullptr) return fail(H3B_EINVAL, "%s: null pointer", what);
  if (stride_x < 0 || s_row < 0 || s_blk < 0) return fail(H3B_EINVAL, "%s: negative stride", what);
  const int64_t KB = (K + BLK - 1) / BLK;
  if (rows > ((1ll << 31) - 1) / KB) return fail(H3B_EUNSUPPORTED, "%s: 2^31 blocks or more", what);
  const bool vec = K % 8 == 0 && stride_x % 8 == 0 && aligned(x, 16) && aligned(q, 8);
  const auto units = static_cast<uint32_t>((rows + 2 * U - 1) / (2 * U) * KB);
  const unsigned grid = (units + 3) / 4;
  const auto* xx = static_cast<const uint16_t*>(x);
  auto* qq = static_cast<uint8_t*>(q);
  return launch(what, vec ? quant_blocks_kernel<true, SILU> : quant_blocks_kernel<false, SILU>, grid, 128, st, xx,
                static_cast<uint32_t>(rows), units, static_cast<uint32_t>(KB), K, stride_x, qq, s, s_row, s_blk,
                static_cast<int>(div_mode));
}

}  // namespace
}  // namespace h3b

using namespace h3b;

extern "C" int h3b_quant_blocks_e4m3(const void* x, int64_t rows, int64_t cols, int64_t stride_x, void* q, float* scale,
                                     int64_t scale_row, int64_t scale_block, int32_t div_mode, h3b_stream_t stream) {
  return quant_blocks<false>("quant_blocks", x, rows, cols, stride_x, q, scale, scale_row, scale_block, div_mode,
                             reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int h3b_silu_mul_quant_blocks_e4m3(const void* x, int64_t rows, int64_t d, int64_t stride_x, void* q,
                                              float* scale, int64_t scale_row, int64_t scale_block, int32_t div_mode,
                                              h3b_stream_t stream) {
  return quant_blocks<true>("silu_mul_quant_blocks", x, rows, d, stride_x, q, scale, scale_row, scale_block, div_mode,
                            reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int h3b_quant_weight_blocks_e4m3(const void* w, int64_t experts, int64_t n, int64_t k, int64_t stride_e,
                                            int64_t stride_n, void* q, float* scale, int32_t div_mode,
                                            h3b_stream_t stream) {
  if (experts < 0 || n < 0 || k < 0)
    return fail(H3B_EINVAL, "quant_weight_blocks: experts %lld n %lld k %lld", (long long)experts, (long long)n,
                (long long)k);
  if (bad_mode(div_mode)) return fail(H3B_EINVAL, "quant_weight_blocks: div_mode %d", div_mode);
  if (experts == 0 || n == 0 || k == 0) return H3B_OK;
  if (w == nullptr || q == nullptr || scale == nullptr) return fail(H3B_EINVAL, "quant_weight_blocks: null pointer");
  if (stride_e < 0 || stride_n < 0) return fail(H3B_EINVAL, "quant_weight_blocks: negative stride");
  const int64_t NB = (n + BLK - 1) / BLK, KB = (k + BLK - 1) / BLK, most = (1ll << 31) - 1;
  if (NB > most / KB || experts > most / (NB * KB)) return fail(H3B_EUNSUPPORTED, "quant_weight_blocks: 2^31 tiles or more");
  const bool vec = k % 8 == 0 && stride_n % 8 == 0 && stride_e % 8 == 0 && aligned(w, 16) && aligned(q, 8);
  const unsigned grid = static_cast<unsigned>(experts * NB * KB);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto* ww = static_cast<const uint16_t*>(w);
  auto* qq = static_cast<uint8_t*>(q);
  return launch("quant_weight_blocks", vec ? quant_weight_blocks_kernel<true> : quant_weight_blocks_kernel<false>, grid,
                256, st, ww, n, k, stride_e, stride_n, static_cast<uint32_t>(NB), static_cast<uint32_t>(KB), qq, scale,
                static_cast<int>(div_mode));
}
