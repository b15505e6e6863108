// Block-scaled FP8 quantisation (HBM bound): e4m3 values with one fp32 scale for each 128 consecutive values of a row
// (activations; plain, or of silu(gate) * up) or for each 128 x 128 tile (weights).  The scale and the rounding are
// those of the per-token quant, taken over a block:
//   scale = max(amax / 448, 1/(448*512)),  q = e4m3_rn(clamp(h * (1 / scale), -448, 448))     (NaN propagates)
//
// Activations: eight lanes hold a block, 16 values each in one 32-byte load, reduce its abs-max by shuffles and write 16 bytes
// of e4m3 a lane; no shared memory, no barrier.  A warp takes the same block of eight consecutive rows (blocks taken along a
// row instead, each with divisions and a 4-byte scale store of its own, ran at 4.9 TB/s).  Weights: a CTA of 256 threads
// holds a 128 x 128 tile in registers and reduces it once (512 threads: 50 us for 36).  Every value is read once and
// written once.
//
// Long runs sit at the power cap, where each instruction costs clock, so their number counts although memory bounds the
// kernels: 62,496 x 5,120 takes 142 us, 6.8 TB/s (a plain copy of as many bytes 148); silu-mul, 31,248 x 13,824, 320 to 332 us
// on different days, 6.6 to 6.8 TB/s; weight 15,360 x 5,120 36 us, 6.5 TB/s.  With 16-byte loads 153, 362 and 36 us; with
// checks and 64-bit products for every load and single instead of packed fp32 products, twice the instructions, 168, 401 and
// 39 us.  Load and store hints (evict first, no allocation in L1) measure the same or slower.
#include "common.cuh"
#include "quant.cuh"

namespace h3b {
namespace {

constexpr int BLK = 128;

// 16 bf16 values as bit patterns
struct V16 {
  uint32_t w[8];
};

// How a lane's 16 values of a block move: one 32-byte load and one 16-byte store, two 16-byte loads and 8-byte stores, or
// value by value, every eighth from the lane's (its neighbours take the ones between: 999 x 5,130 in 25 us with 16 in a row)
enum { SCALAR = 0, VEC16 = 1, VEC32 = 2 };
template <int MODE>
__device__ __forceinline__ int first_column() {
  return (threadIdx.x & 7) * (MODE == SCALAR ? 1 : 16);
}

// 16 values at x, `left` columns before the row's end; those past it as zero.  ALL: every one is in the row.  VEC32: K % 16 ==
// 0, so all 16 are in the row or past it, VEC16: K % 8 == 0.  Plain loads: the kernel ahead may write x while this one already
// runs (common.cuh).
template <int MODE, bool ALL>
__device__ __forceinline__ V16 load16(const uint16_t* x, int64_t left) {
  V16 v = {};
  if constexpr (MODE == VEC32) {
    if (ALL || left > 0)
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]),
                     "=r"(v.w[7])
                   : "l"(x));
  } else if constexpr (MODE == VEC16) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!ALL && left <= 8 * h) continue;
      const uint4 a = reinterpret_cast<const uint4*>(x)[h];
      v.w[4 * h] = a.x;
      v.w[4 * h + 1] = a.y;
      v.w[4 * h + 2] = a.z;
      v.w[4 * h + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = 16 * i < left ? x[16 * i] : 0u;
      const uint32_t hi = 16 * i + 8 < left ? x[16 * i + 8] : 0u;
      v.w[i] = lo | (hi << 16);
    }
  }
  return v;
}

template <int MODE, bool ALL>
__device__ __forceinline__ void store16(uint8_t* q, int64_t left, uint4 v) {
  if constexpr (MODE == VEC32) {
    if (ALL || left > 0) *reinterpret_cast<uint4*>(q) = v;
  } else if constexpr (MODE == VEC16) {
    if (ALL || left > 0) *reinterpret_cast<uint2*>(q) = make_uint2(v.x, v.y);
    if (ALL || left > 8) *reinterpret_cast<uint2*>(q + 8) = make_uint2(v.z, v.w);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (8 * i < left) q[8 * i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
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
__device__ __forceinline__ uint32_t absmax_of(const V16& v) {
  return absmax2(absmax2(absmax2(v.w[0], v.w[1]), absmax2(v.w[2], v.w[3])),
                 absmax2(absmax2(v.w[4], v.w[5]), absmax2(v.w[6], v.w[7])));
}
// the bits of a bf16 magnitude as those of an fp32 (they order like the magnitudes, NaN above all)
__device__ __forceinline__ uint32_t absmax_bits(uint32_t m2) { return fold16(m2 & 0x7FFF7FFFu) << 16; }

// x * inv to e4m3, to nearest even; satfinite clamps to +-448 and keeps NaN
__device__ __forceinline__ uint4 quant16(const F2 (&x)[8], float inv) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 a = mul2(x[2 * i], F2{inv, inv}), b = mul2(x[2 * i + 1], F2{inv, inv});
    o[i] = static_cast<uint32_t>(f32x2_to_e4m3x2(a.lo, a.hi)) | (static_cast<uint32_t>(f32x2_to_e4m3x2(b.lo, b.hi)) << 16);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ uint4 quant16_bf16(const V16& v, float inv) {
  F2 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = unpack2(v.w[i]);
  return quant16(x, inv);
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits, int div_mode) {
  return nan_max(qdiv(__uint_as_float(amax_bits), kFp8Max, div_mode), kMinScale);
}

// silu(g) * u = g / (1 + 2^(-g log2 e)) * u in fp32, not rounded before the quant: one rounding, to e4m3.  The argument's
// rounding counts |g| * 0.75, ex2.approx 2, rcp.approx 1 and the other four steps half a unit each: within (5 + 0.75 |g|) *
// 2^-23 in all (g and the result being normal numbers), against the 2^-4 of e4m3.  For gates down to -87: below, the reciprocal
// is under 2^-126 and flushed.
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

// The same for any gate: below -87, silu(g) = g 2^(g log2 e) to 2^-125, computed 2^64 times as large and scaled back behind the
// product with u, which may be 2^127.  Within the same bound.  (From g = -131 on the exponential is flushed even so, and |h| is
// under 10^-16: a code of 0.)  -inf gives NaN, as g / (1 + exp(-g)) does.
__device__ __forceinline__ float silu_mul_far(float g, float u) {
  const F2 near = silu_mul2(F2{g, g}, F2{u, u});
  float e = fmaf(g, 1.4426950408889634f, 64.0f);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e));
  return g < -87.0f ? g * e * u * 5.421010862427522e-20f : near.lo;
}

constexpr int U = 2, ROWS = 4 * U;  // rows of a lane (eight lanes hold a block), rows of a warp

// Whether a warp's gates have one below -87 and its ups one of 2^90 or more (or either a NaN).  With smaller ups silu(g) * u of
// such a gate is under 2^-29: a code of 0 by either way, and nothing to the block's maximum.  As unsigned 16-bit patterns the
// negative gates lie above the others, in the order of their magnitudes.
__device__ __forceinline__ bool any_far(const V16 (&gate)[U], const V16 (&up)[U]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vimax3_u16x2(m, gate[0].w[i], gate[1].w[i]);
  if (!__any_sync(0xffffffffu, fold16(m) > 0xC2AEu)) return false;
  m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vimax3_u16x2(m, up[0].w[i] & 0x7FFF7FFFu, up[1].w[i] & 0x7FFF7FFFu);
  return __any_sync(0xffffffffu, fold16(m) >= 0x6C80u);
}

// A unit (as below) with such values, which hardly ever come up: value by value, `step` columns apart, each twice, in few
// registers.  A call, so that the other units' code stays as it is: with both in one loop 31,248 x 13,824 takes 6 % longer
// (nothing measurable so; 2 ms for 300 us if every unit has such values).
__device__ __noinline__ void far_unit(const uint16_t* x, int64_t stride_x, int64_t K, int rows, int64_t left, int step,
                                      uint8_t* q, float* s, int64_t s_row, int div_mode) {
  auto value = [&](int i) {
    return silu_mul_far(bf16_bits_to_f32(x[step * i]), bf16_bits_to_f32(x[K + step * i]));
  };
#pragma unroll 1
  for (int u = 0; u < U; ++u, x += stride_x, q += K, s += s_row) {
    float m = 0.0f;
#pragma unroll 1
    for (int i = 0; i < 16 && u < rows && step * i < left; ++i)
      asm("max.NaN.abs.f32 %0, %0, %1, 0f00000000;" : "+f"(m) : "f"(value(i)));
    uint32_t amax = __float_as_uint(m);
#pragma unroll
    for (int o = 4; o; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = block_scale(amax, div_mode);
    const float inv = qdiv(1.0f, scale, div_mode);
    if ((threadIdx.x & 7) == 0 && u < rows) *s = scale;
#pragma unroll 1
    for (int i = 0; i < 16 && u < rows && step * i < left; ++i)
      q[step * i] = static_cast<uint8_t>(f32x2_to_e4m3x2(value(i) * inv, 0.0f));
  }
}

// A warp's unit: one block of ROWS consecutive rows, at x the lane's first row and column (SILU: up columns K further on).
// `rows`, `left`: rows from the lane's first and columns from the lane's first to the end.
template <int MODE, bool SILU, bool ALL>
__device__ __forceinline__ void quant_unit(const uint16_t* x, int64_t stride_x, int64_t K, int rows,
                                           int64_t left, uint8_t* __restrict__ q, float* __restrict__ s, int64_t s_row,
                                           int div_mode) {
  static_assert(U == 2, "a lane's two rows");
  constexpr uint32_t FULL = 0xffffffffu;
  V16 v[U], w[SILU ? U : 1];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    v[u] = V16{};
    if (SILU) w[u] = V16{};
    if (ALL || u < rows) {
      v[u] = load16<MODE, ALL>(x, left);
      if (SILU) w[u] = load16<MODE, ALL>(x + K, left);
    }
    x += stride_x;
  }
  if constexpr (SILU) {
    if (any_far(v, w))  // the whole warp
      return far_unit(x - U * stride_x, stride_x, K, rows, left, MODE == SCALAR ? 8 : 1, q, s, s_row, div_mode);
  }
  // each lane is left with the largest magnitude of its row `mine` over the eight lanes, as fp32 bits
  const bool mine = threadIdx.x & 4;
  F2 y[SILU ? U : 1][8];
  uint32_t amax;
  if constexpr (SILU) {
    float m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[u][e] = silu_mul2(unpack2(v[u].w[e]), unpack2(w[u].w[e]));
        asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m[u]) : "f"(y[u][e].lo), "f"(y[u][e].hi));
      }
    }
    const uint32_t a = __float_as_uint(m[0]), b = __float_as_uint(m[1]);
    amax = max(mine ? b : a, __shfl_xor_sync(FULL, mine ? a : b, 4));
    amax = max(amax, __shfl_xor_sync(FULL, amax, 2));
    amax = max(amax, __shfl_xor_sync(FULL, amax, 1));
  } else {
    // both rows' maxima as one pair of 16 bits
    const uint32_t a = absmax_of(v[0]), b = absmax_of(v[1]);
    uint32_t m2 = absmax2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632)) & 0x7FFF7FFFu;
#pragma unroll
    for (int o = 4; o; o >>= 1) m2 = __vmaxu2(m2, __shfl_xor_sync(FULL, m2, o));
    amax = mine ? m2 & 0xFFFF0000u : m2 << 16;
  }
  const float scale = block_scale(amax, div_mode);
  const float inv = qdiv(1.0f, scale, div_mode);
  if ((threadIdx.x & 3) == 0 && (ALL || static_cast<int>(mine) < rows)) *(mine ? s + s_row : s) = scale;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv_u = __shfl_sync(FULL, inv, (threadIdx.x & 24) + 4 * u);
    if (ALL || u < rows) {
      if constexpr (SILU)
        store16<MODE, ALL>(q, left, quant16(y[u], inv_u));
      else
        store16<MODE, ALL>(q, left, quant16_bf16(v[u], inv_u));
    }
    q += K;
  }
}

// rows x [rows, K] (SILU: [rows, 2K], gate | up) -> q [rows, K], s[row * s_row + j * s_blk].  A warp takes block j of ROWS
// consecutive rows: their scales are then neighbours in the block-major scale tensor and leave in one store, each division
// is made once per warp for all of them, and the loads of a CTA's 4 warps run along the rows.  KB_inv: 2^64 / KB rounded up
// (0 for KB = 1), so that a 64-bit product's upper half divides any 32-bit number by KB.
template <int MODE, bool SILU>
__global__ void __launch_bounds__(128) quant_blocks_kernel(const uint16_t* x, uint32_t rows, uint32_t units,
                                                           uint32_t KB, uint64_t KB_inv, int64_t K, int64_t stride_x,
                                                           uint8_t* __restrict__ q, float* __restrict__ s, int64_t s_row,
                                                           int64_t s_blk, int div_mode) {
  pdl_wait();
  pdl_launch();
  const uint32_t unit = blockIdx.x * 4u + (threadIdx.x >> 5);
  if (unit >= units) return;  // the whole warp
  const uint32_t group = KB_inv ? static_cast<uint32_t>(__umul64hi(KB_inv, unit)) : unit, j = unit - group * KB;
  const int64_t row0 = static_cast<int64_t>(group) * ROWS + (threadIdx.x >> 3 & 3) * U;
  const int64_t c = static_cast<int64_t>(j) * BLK + first_column<MODE>();
  x += row0 * stride_x + c;
  q += row0 * K + c;
  s += row0 * s_row + j * s_blk;
  if (MODE != SCALAR && (group + 1) * ROWS <= rows && (j + 1) * static_cast<int64_t>(BLK) <= K)
    quant_unit<MODE, SILU, MODE != SCALAR>(x, stride_x, K, U, 16, q, s, s_row, div_mode);
  else
    quant_unit<MODE, SILU, false>(x, stride_x, K, static_cast<int>(rows) - static_cast<int>(row0), K - c, q, s, s_row,
                                  div_mode);
}

// A CTA's tile: rows r0 + 32 u (u < 4) of the lane at w, step_w elements apart, 16 columns each.  `rows`, `left` as above.
template <int MODE, bool ALL>
__device__ __forceinline__ void quant_tile(const uint16_t* w, int64_t step_w, int64_t rows, int64_t left,
                                           uint8_t* __restrict__ q, int64_t step_q, float* __restrict__ s, int div_mode) {
  __shared__ uint32_t red[8];
  __shared__ float tile_scale[2];  // and its inverse
  V16 v[4];
  uint32_t m2 = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    v[u] = V16{};
    if (ALL || 32 * u < rows) v[u] = load16<MODE, ALL>(w, left);
    w += step_w;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) m2 = absmax2(m2, absmax_of(v[u]));
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
  for (int u = 0; u < 4; ++u) {
    if (ALL || 32 * u < rows) store16<MODE, ALL>(q, left, quant16_bf16(v[u], inv));
    q += step_q;
  }
}

// w [E, N, K] -> q [E, N, K] contiguous, s [E, NB, KB] contiguous: one CTA per tile
template <int MODE>
__global__ void __launch_bounds__(256) quant_weight_blocks_kernel(const uint16_t* w, int64_t N, int64_t K,
                                                                  int64_t stride_e, int64_t stride_n, uint32_t NB,
                                                                  uint32_t KB, uint8_t* __restrict__ q,
                                                                  float* __restrict__ s, int div_mode) {
  pdl_wait();
  pdl_launch();
  const uint32_t tile = blockIdx.x;
  const uint32_t j = tile % KB, en = tile / KB, i = en % NB, e = en / NB;
  const int64_t c = static_cast<int64_t>(j) * BLK + first_column<MODE>();
  const int64_t r0 = static_cast<int64_t>(i) * BLK + (threadIdx.x >> 3);
  w += e * stride_e + r0 * stride_n + c;
  q += (e * N + r0) * K + c;
  s += tile;
  if (MODE != SCALAR && (i + 1) * static_cast<int64_t>(BLK) <= N && (j + 1) * static_cast<int64_t>(BLK) <= K)
    quant_tile<MODE, MODE != SCALAR>(w, 32 * stride_n, BLK, 16, q, 32 * K, s, div_mode);
  else
    quant_tile<MODE, false>(w, 32 * stride_n, N - r0, K - c, q, 32 * K, s, div_mode);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// how rows of K values at x (strides in elements) and bytes at q move
int mode(const void* x, int64_t K, int64_t stride, int64_t stride2, const void* q) {
  if (K % 16 == 0 && stride % 16 == 0 && stride2 % 16 == 0 && aligned(x, 32) && aligned(q, 16)) return VEC32;
  return K % 8 == 0 && stride % 8 == 0 && stride2 % 8 == 0 && aligned(x, 16) && aligned(q, 8) ? VEC16 : SCALAR;
}

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
  const auto units = static_cast<uint32_t>((rows + ROWS - 1) / ROWS * KB);
  const unsigned grid = (units + 3) / 4;
  const int m = mode(x, K, stride_x, 0, q);
  const auto kernel = m == VEC32 ? quant_blocks_kernel<VEC32, SILU>
                                 : (m == VEC16 ? quant_blocks_kernel<VEC16, SILU> : quant_blocks_kernel<SCALAR, SILU>);
  return launch(what, kernel, grid, 128, st, static_cast<const uint16_t*>(x), static_cast<uint32_t>(rows), units,
                static_cast<uint32_t>(KB), KB > 1 ? ~0ull / static_cast<uint64_t>(KB) + 1 : 0ull, K, stride_x,
                static_cast<uint8_t*>(q), s, s_row, s_blk, static_cast<int>(div_mode));
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
  const unsigned grid = static_cast<unsigned>(experts * NB * KB);
  const int m = mode(w, k, stride_n, stride_e, q);
  const auto kernel = m == VEC32 ? quant_weight_blocks_kernel<VEC32>
                                 : (m == VEC16 ? quant_weight_blocks_kernel<VEC16> : quant_weight_blocks_kernel<SCALAR>);
  return launch("quant_weight_blocks", kernel, grid, 256, reinterpret_cast<cudaStream_t>(stream),
                static_cast<const uint16_t*>(w), n, k, stride_e, stride_n, static_cast<uint32_t>(NB),
                static_cast<uint32_t>(KB), static_cast<uint8_t*>(q), scale, static_cast<int>(div_mode));
}
