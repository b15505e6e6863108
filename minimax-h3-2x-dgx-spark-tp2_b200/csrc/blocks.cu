// Block-scaled FP8 quantisation (HBM bound): e4m3 values with one fp32 scale for each 128 consecutive values of a row
// (activations; plain, or of silu(gate) * up) or for each 128 x 128 tile (weights).  The scale and the rounding are
// those of the per-token quant, taken over a block:
//   scale = max(amax / 448, 1/(448*512)),  q = e4m3_rn(clamp(h * (1 / scale), -448, 448))     (NaN propagates)
//
// Activations: 16 lanes hold a block as one 16-byte load each (8 bf16 values), reduce its abs-max inside the half-warp and
// write 128 bytes of e4m3; no shared memory, no barrier.  A warp takes the same block of eight consecutive rows (blocks taken
// along a row instead, each with divisions and a 4-byte scale store of its own, ran at 4.9 TB/s).  Weights: a CTA of 256
// threads holds a 128 x 128 tile in registers (8 vectors per thread) and reduces it once (512 threads: 50 us for 36).  Every
// value is read once and written once.
//
// Measured in long runs, which sit at the power cap (1.6 GHz): 62,496 x 5,120 in 153 us, 6.3 TB/s (139 us before the cap
// sets in; a plain copy of as many bytes 148, under the cap); silu-mul, 31,248 x 13,824, 362 us, 6.0 TB/s (312 before); weight
// 15,360 x 5,120 in 36 us.  Instructions are what the power goes into: with about twice as many the same calls took 168, 401
// and 39 us.  Load and store hints (evict first, no allocation in L1) measure the same or slower.
#include "common.cuh"
#include "quant.cuh"

namespace h3b {
namespace {

constexpr int BLK = 128;

// 8 bf16 values at x, `left` columns before the row's end, as bit patterns.  ALL: every one is in the row.  VEC: one 16-byte
// load (K % 8 == 0, so they are all in the row or all past it); otherwise value by value, those past the end as zero
template <bool VEC, bool ALL>
__device__ __forceinline__ uint4 load8(const uint16_t* x, int64_t left) {
  if constexpr (VEC) {
    return ALL || left > 0 ? __ldg(reinterpret_cast<const uint4*>(x)) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < left ? x[2 * i] : 0u;
      const uint32_t hi = 2 * i + 1 < left ? x[2 * i + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <bool VEC, bool ALL>
__device__ __forceinline__ void store8(uint8_t* q, int64_t left, uint2 v) {
  if constexpr (VEC) {
    if (ALL || left > 0) *reinterpret_cast<uint2*>(q) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) q[i] = static_cast<uint8_t>((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
  }
}

// Two fp32 operations per instruction.  The large calls run at the power cap, where instructions cost clock: with these, the
// pointers stepped from row to row and the checks of whole blocks made once, the quantisers issue half as many.
struct F2 {
  float lo, hi;
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.lo), "=f"(r.hi)
      : "f"(a.lo), "f"(a.hi), "f"(b.lo), "f"(b.hi));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.lo), "=f"(r.hi)
      : "f"(a.lo), "f"(a.hi), "f"(b.lo), "f"(b.hi));
  return r;
}
__device__ __forceinline__ F2 unpack2(uint32_t w) { return F2{lo_bf16(w), hi_bf16(w)}; }

// larger magnitudes of two bf16 pairs (signs: anything; NaN if either is)
__device__ __forceinline__ uint32_t absmax2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t absmax_of(const uint4& v) { return absmax2(absmax2(v.x, v.y), absmax2(v.z, v.w)); }
// the largest magnitude of a pair, as the bits of an fp32 (they order like the magnitudes, NaN above all)
__device__ __forceinline__ uint32_t absmax_bits(uint32_t m2) { return fold16(m2 & 0x7FFF7FFFu) << 16; }

// x * inv to e4m3, to nearest even; satfinite clamps to +-448 and keeps NaN
__device__ __forceinline__ uint2 quant8(const F2 (&x)[4], float inv) {
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 a = mul2(x[2 * i], F2{inv, inv}), b = mul2(x[2 * i + 1], F2{inv, inv});
    o[i] = static_cast<uint32_t>(f32x2_to_e4m3x2(a.lo, a.hi)) | (static_cast<uint32_t>(f32x2_to_e4m3x2(b.lo, b.hi)) << 16);
  }
  return make_uint2(o[0], o[1]);
}
__device__ __forceinline__ uint2 quant8_bf16(const uint4& v, float inv) {
  const F2 x[4] = {unpack2(v.x), unpack2(v.y), unpack2(v.z), unpack2(v.w)};
  return quant8(x, inv);
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits, int div_mode) {
  return nan_max(qdiv(__uint_as_float(amax_bits), kFp8Max, div_mode), kMinScale);
}

// silu(g) * u = g / (1 + 2^(-g log2 e)) * u in fp32, not rounded before the quant: one rounding, to e4m3.  The argument's
// rounding counts |g| * 0.75, ex2.approx 2, rcp.approx 1 and the other four steps half a unit each: within (5 + 0.75 |g|) *
// 2^-23 in all, against the 2^-4 of e4m3.  Below g = -87 the reciprocal, under 2^-126, is flushed and silu is 0.
__device__ __forceinline__ F2 silu_mul2(F2 g, F2 u) {
  constexpr float NEG_LOG2E = -1.4426950408889634f;
  F2 e = mul2(g, F2{NEG_LOG2E, NEG_LOG2E});
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.lo));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.hi));
  F2 r = add2(e, F2{1.0f, 1.0f});
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.lo));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.hi));
  return mul2(mul2(g, r), u);
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

// A warp's unit: blocks of 2U consecutive rows at x (the lane's first row and column; SILU: up columns `K` further on), of
// which this lane's half-warp has U.  `rows`, `left`: rows from the lane's first and columns from the lane's first to the end.
template <bool VEC, bool SILU, bool ALL>
__device__ __forceinline__ void quant_unit(const uint16_t* __restrict__ x, int64_t stride_x, int64_t K, int rows,
                                           int64_t left, uint8_t* __restrict__ q, float* __restrict__ s, int64_t s_row,
                                           int div_mode) {
  const int hl = threadIdx.x & 15;
  uint4 v[U], w[SILU ? U : 1];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    v[u] = make_uint4(0, 0, 0, 0);
    if (SILU) w[u] = make_uint4(0, 0, 0, 0);
    if (ALL || u < rows) {
      v[u] = load8<VEC, ALL>(x, left);
      if (SILU) w[u] = load8<VEC, ALL>(x + K, left);
    }
    x += stride_x;
  }
  F2 y[SILU ? U : 1][4];
  uint32_t amax[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if constexpr (SILU) {
      const uint32_t g[4] = {v[u].x, v[u].y, v[u].z, v[u].w}, up[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      float m = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[u][e] = silu_mul2(unpack2(g[e]), unpack2(up[e]));
        asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(y[u][e].lo), "f"(y[u][e].hi));
      }
      amax[u] = __float_as_uint(m);
    } else {
      amax[u] = absmax_bits(absmax_of(v[u]));
    }
  }
  const float scale = block_scale(half_warp_max(amax, hl), div_mode);
  const float inv = qdiv(1.0f, scale, div_mode);
  if (hl % 4 == 0 && (ALL || hl / 4 < rows)) s[hl / 4 * s_row] = scale;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv_u = __shfl_sync(0xffffffffu, inv, (threadIdx.x & 16) + u * 4);
    if (ALL || u < rows) {
      if constexpr (SILU)
        store8<VEC, ALL>(q, left, quant8(y[u], inv_u));
      else
        store8<VEC, ALL>(q, left, quant8_bf16(v[u], inv_u));
    }
    q += K;
  }
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
  const uint32_t unit = blockIdx.x * 4u + (threadIdx.x >> 5);
  if (unit >= units) return;  // the whole warp
  const uint32_t group = unit / KB, j = unit - group * KB;
  const int64_t row0 = static_cast<int64_t>(group) * (2 * U) + (threadIdx.x & 16 ? U : 0);
  const int64_t c = static_cast<int64_t>(j) * BLK + (threadIdx.x & 15) * 8;
  x += row0 * stride_x + c;
  q += row0 * K + c;
  s += row0 * s_row + j * s_blk;
  const bool all = (group + 1) * (2 * U) <= rows && (j + 1) * static_cast<int64_t>(BLK) <= K;
  if (VEC && all)
    quant_unit<VEC, SILU, VEC>(x, stride_x, K, U, 8, q, s, s_row, div_mode);
  else
    quant_unit<VEC, SILU, false>(x, stride_x, K, static_cast<int>(rows) - static_cast<int>(row0), K - c, q, s, s_row,
                                 div_mode);
}

// A CTA's tile: rows tile row r0 + 16 u of the lane at w (step_w elements apart), 8 columns each.  `rows`, `left` as above.
template <bool VEC, bool ALL>
__device__ __forceinline__ void quant_tile(const uint16_t* __restrict__ w, int64_t step_w, int64_t rows, int64_t left,
                                           uint8_t* __restrict__ q, int64_t step_q, float* __restrict__ s, int div_mode) {
  __shared__ uint32_t red[8];
  __shared__ float tile_scale[2];  // and its inverse
  uint4 v[8];
  uint32_t m2 = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    v[u] = ALL || 16 * u < rows ? load8<VEC, ALL>(w, left) : make_uint4(0, 0, 0, 0);
    m2 = absmax2(m2, absmax_of(v[u]));
    w += step_w;
  }
  const uint32_t wmax = __reduce_max_sync(0xffffffffu, absmax_bits(m2));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = wmax;
  __syncthreads();
  uint32_t amax = red[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) amax = max(amax, red[k]);
  if (threadIdx.x < 32) {  // the divisions in one warp: in all eight they took a tenth of the kernel
    const float scale = block_scale(amax, div_mode);
    tile_scale[0] = scale;
    tile_scale[1] = qdiv(1.0f, scale, div_mode);
  }
  __syncthreads();
  const float inv = tile_scale[1];
  if (threadIdx.x == 0) *s = tile_scale[0];  // behind the barrier: ahead of it the others waited for it, 39.4 us for 36
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    if (ALL || 16 * u < rows) store8<VEC, ALL>(q, left, quant8_bf16(v[u], inv));
    q += step_q;
  }
}

// w [E, N, K] -> q [E, N, K] contiguous, s [E, NB, KB] contiguous: one CTA per tile
template <bool VEC>
__global__ void __launch_bounds__(256) quant_weight_blocks_kernel(const uint16_t* __restrict__ w, int64_t N, int64_t K,
                                                                  int64_t stride_e, int64_t stride_n, uint32_t NB,
                                                                  uint32_t KB, uint8_t* __restrict__ q,
                                                                  float* __restrict__ s, int div_mode) {
  pdl_wait();
  pdl_launch();
  const uint32_t tile = blockIdx.x;
  const uint32_t j = tile % KB, en = tile / KB, i = en % NB, e = en / NB;
  const int64_t c = static_cast<int64_t>(j) * BLK + (threadIdx.x & 15) * 8;
  const int64_t r0 = static_cast<int64_t>(i) * BLK + (threadIdx.x >> 4);
  w += e * stride_e + r0 * stride_n + c;
  q += (e * N + r0) * K + c;
  s += tile;
  if (VEC && (i + 1) * static_cast<int64_t>(BLK) <= N && (j + 1) * static_cast<int64_t>(BLK) <= K)
    quant_tile<VEC, VEC>(w, 16 * stride_n, BLK, 8, q, 16 * K, s, div_mode);
  else
    quant_tile<VEC, false>(w, 16 * stride_n, N - r0, K - c, q, 16 * K, s, div_mode);
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
