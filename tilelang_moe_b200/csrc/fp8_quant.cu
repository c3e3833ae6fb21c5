// 8-bit operands: e4m3 values with an fp32 scale per 128 elements of a row, or per 128 x 128 block of a weight.
//
//   top   = max(max |x| over the group, 2^-100)        NaN where the group holds one
//   scale = top / 448                                   448 is the largest e4m3 number
//   q     = e4m3(x * (448 / top))                       to nearest, ties to even
//
// so that q * scale is x to within half an e4m3 step.  A group of zeros has the scale 2^-100 / 448, never 0; a group with an
// infinity or a NaN comes out as NaN in its places, or all of it.  The same for x = SiLU(gate) * up, computed in fp32 and never
// rounded to 16 bits in between.
//
// Bound by memory: an element is read once (2 or 4 bytes, twice that for SiLU) and written once (1 byte), and the group's
// maximum is taken on the registers that its values stay in.
#include "vec.cuh"

namespace moe {
namespace fp8 {

constexpr int G = 128;               // elements that share a scale along a row
constexpr float TOP = 448.0f;
constexpr uint32_t TINY_BITS = 0x0D800000u;   // 2^-100: 448 / top and top / 448 stay normal numbers

// two fp32 -> two e4m3 in 16 bits, the first in the lower byte
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
template <int N>
__device__ __forceinline__ Raw<N> quantize(const float* x, float inv) {
  if constexpr (N == 1) return (uint8_t)e4m3x2(x[0] * inv, 0.f);
  else if constexpr (N == 2) return (uint16_t)e4m3x2(x[0] * inv, x[1] * inv);
  else if constexpr (N == 4) return e4m3x2(x[0] * inv, x[1] * inv) | (e4m3x2(x[2] * inv, x[3] * inv) << 16);
  else {
    uint2 o;
    o.x = quantize<4>(x, inv);
    o.y = quantize<4>(x + 4, inv);
    return o;
  }
}
// max(m, |x|), NaN where either is one
__device__ __forceinline__ float max_magnitude(float m, float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(x)));
  return m;
}
// The largest of a group's magnitudes is the largest of their bits: no sign, every NaN above infinity.
__device__ __forceinline__ float group_top(uint32_t bits) { return __uint_as_float(max(bits, TINY_BITS)); }

// 448 / top and top / 448, each from an approximate quotient and its remainder in one fma (Markstein, IBM J. Res. Dev. 34, 1990);
// an infinite top has no remainder, and the first quotients, 0 and infinity, stand.  The checked divisions cost as much as
// the rest of a group: 8192 x 7168 bf16 38.5 -> 36.0 us with both and the maximum by max.NaN.
__device__ __forceinline__ float inverse_of(float top) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(top));
  const float q = TOP * y, rem = fmaf(-top, q, TOP);
  return fabsf(rem) >= 0.f ? fmaf(rem, y, q) : q;
}
__device__ __forceinline__ float scale_of(float top) {
  constexpr float r = 1.0f / TOP;
  const float q = top * r, rem = fmaf(-TOP, q, top);
  return fabsf(rem) >= 0.f ? fmaf(rem, r, q) : q;
}

// g * sigmoid(g) * u to within 2^-21, because the scale of a group shows what its 8-bit values do not.  The quotient is an approximate
// one and its remainder, on a quarter of both operands: the reciprocal of the largest sums would be flushed to zero.  The
// remainder is NaN where gate or sum is infinite: the first quotient stands.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float d4 = fmaf(expf(-g), 0.25f, 0.25f), g4 = 0.25f * g;
  float r4;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r4) : "f"(d4));
  const float q = g4 * r4, rem4 = fmaf(-d4, q, g4);
  return (fabsf(rem4) > 0.0f ? fmaf(rem4, r4, q) : q) * u;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// The same for the elements of a vector, into g.  Gates up to 80, where nothing overflows, two at a time: exp(-g) = 2^h exp(-s) with
// h = -g / ln 2 rounded and s = g + h ln 2, ln 2 in two parts (Cody and Waite, 1980), exp(-s) = 1 - s for an s below 2^-16.  Issue
// slots count in this form of the kernel, 65 % of them are taken; 32769 x 2048 bf16, states in turn: expf for every gate 71.3 us,
// this 62.5 (with the fast exponential and without the remainder, off by 1.0e-6 at gates of -20 and 3.8e-6 at -80, 59.7).
template <int N>
__device__ __forceinline__ void silu_mul(float (&g)[N], const float (&u)[N]) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = max_magnitude(top, g[j]);
  if (N % 2 == 0 && top <= 80.0f) {
#pragma unroll
    for (int j = 0; j + 1 < N; j += 2) {
      const float2 g2 = make_float2(g[j], g[j + 1]);
      const float2 h = mul2(g2, both(-1.44269504088896341f));
      const float2 s = fma2(h, both(-1.90465429995776769e-9f), fma2(h, both(0.693147182464599609f), g2));
      float2 e, r;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(h.x));
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(h.y));
      const float2 minus_d = fma2(e, fma2(s, both(1.0f), both(-1.0f)), both(-1.0f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(-minus_d.x));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(-minus_d.y));
      const float2 q = mul2(g2, r);
      const float2 o = mul2(fma2(fma2(minus_d, q, g2), r, q), make_float2(u[j], u[j + 1]));
      g[j] = o.x;
      g[j + 1] = o.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) g[j] = silu_mul(g[j], u[j]);
  }
}

struct RowParams {
  const void* x;         // or the gate
  const void* up;
  int64_t x_stride, up_stride;   // elements
  uint32_t groups;       // rows x groups of a row
  int K;                 // elements of a row
  FastDiv per_row;       // groups of a row
  uint8_t* q;
  float* scale;
};

// Two vectors of a group per lane, so that what a group costs beside its elements (the steps to its maximum, the quotients,
// its number) is shared by as many of them: 8192 x 7168 bf16 36.0 -> 30.1 us.  Four vectors of loads in flight per lane, eight
// where they are narrow (rows of odd widths and strides); twice as many were slower (49 us).
template <class T, int V, bool SWIGLU>
struct RowShape {
  static constexpr int N = V / (int)sizeof(T);                  // elements of a vector
  static constexpr int L = V == 16 ? G / (2 * N) : 32;          // lanes of a group
  static constexpr int I = G / (N * L);                         // vectors of a lane and group
  static constexpr int U = (V == 16 ? 4 : 8) / I / (SWIGLU ? 2 : 1);   // groups
  static constexpr int PER_WARP = U * (32 / L);                 // groups of a warp
};

// L lanes hold a group, I vectors of N elements each; a warp takes 32 / L groups side by side, U of them in flight per lane.
// Groups are numbered through all rows, so that short rows fill a warp too.
template <class T, int V, bool SWIGLU>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const RowParams p) {
  using S = RowShape<T, V, SWIGLU>;
  using P = Raw<V>;
  constexpr int N = S::N, L = S::L, I = S::I, U = S::U;
  const int lane = threadIdx.x & 31, in = lane % L;
  const uint32_t first = (blockIdx.x * 8 + (threadIdx.x >> 5)) * S::PER_WARP + lane / L;
  P a[U][I], b[U][I];
  uint32_t row[U];
  int col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t g = first + u * (32 / L);
    row[u] = p.per_row.div(g);
    col[u] = g < p.groups ? (int)(g - row[u] * p.per_row.d) * G + in * N : p.K;
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)row[u] * p.x_stride;
    const T* y = SWIGLU ? reinterpret_cast<const T*>(p.up) + (int64_t)row[u] * p.up_stride : x;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int c = col[u] + i * L * N;
      if (c < p.K) {
        a[u][i] = *reinterpret_cast<const P*>(x + c);
        if (SWIGLU) b[u][i] = *reinterpret_cast<const P*>(y + c);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float x[I][N];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      unpack<T, V>(a[u][i], x[i]);
      if (SWIGLU) {
        float y[N];
        unpack<T, V>(b[u][i], y);
        silu_mul<N>(x[i], y);
      }
      if (col[u] + i * L * N < p.K) {
#pragma unroll
        for (int j = 0; j < N; ++j) m = max_magnitude(m, x[i][j]);
      }
    }
    uint32_t bits = __float_as_uint(m);
    if (L == 32) {
      bits = __reduce_max_sync(0xFFFFFFFFu, bits);
    } else {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xFFFFFFFFu, bits, o));
    }
    const float top = group_top(bits);
    const float inv = inverse_of(top);
    uint8_t* q = p.q + (int64_t)row[u] * p.K;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int c = col[u] + i * L * N;
      if (c < p.K) *reinterpret_cast<Raw<N>*>(q + c) = quantize<N>(x[i], inv);
    }
    const uint32_t g = first + u * (32 / L);
    if (in == 0 && g < p.groups) p.scale[g] = scale_of(top);
  }
}

// One CTA of 256 threads per 128 x 128 block, its values in registers from the one read on.  In a narrow form (V below 16
// bytes, rows of odd widths) a thread holds one element of a half row at a time: same registers, narrower accesses.
template <class T, int V>
__global__ void __launch_bounds__(256)
quantize_blocks_kernel(const T* __restrict__ w, int64_t rows, int K, int row_blocks, int col_blocks, uint8_t* __restrict__ q,
                       float* __restrict__ scale) {
  using P = Raw<V>;
  constexpr int N = V / (int)sizeof(T), COLS = G / N, STEP = 256 / COLS, I = G / STEP;    // vectors per row, rows at a time, vectors per thread
  __shared__ uint32_t part[8];
  const int c = threadIdx.x % COLS, r0 = threadIdx.x / COLS;
  const int64_t blk = blockIdx.x;
  const int64_t e = blk / ((int64_t)row_blocks * col_blocks);
  const int rest = (int)(blk - e * row_blocks * col_blocks);
  const int rb = rest / col_blocks, cb = rest - rb * col_blocks;
  const int col = cb * G + c * N;
  const int64_t base = (e * rows + (int64_t)rb * G) * K + col;
  const int left = (int)(rows - (int64_t)rb * G < G ? rows - (int64_t)rb * G : G);
  P v[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int r = r0 + i * STEP;
    if (r < left && col < K) v[i] = *reinterpret_cast<const P*>(w + base + (int64_t)r * K);
  }
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (r0 + i * STEP < left && col < K) {
      float x[N];
      unpack<T, V>(v[i], x);
#pragma unroll
      for (int j = 0; j < N; ++j) mine = max_magnitude(mine, x[j]);
    }
  uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(mine));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, part[i]);
  const float top = group_top(m), inv = inverse_of(top);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int r = r0 + i * STEP;
    if (r < left && col < K) {
      float x[N];
      unpack<T, V>(v[i], x);
      *reinterpret_cast<Raw<N>*>(q + base + (int64_t)r * K) = quantize<N>(x, inv);
    }
  }
  if (threadIdx.x == 0) scale[blk] = scale_of(top);
}

template <class T, int V, bool SWIGLU>
static void launch_rows(const RowParams& p, cudaStream_t st) {
  const uint32_t per_cta = 8 * RowShape<T, V, SWIGLU>::PER_WARP;
  quantize_rows_kernel<T, V, SWIGLU><<<(p.groups + per_cta - 1) / per_cta, 256, 0, st>>>(p);
}

template <bool SWIGLU>
static int quantize_rows(const void* x, int64_t x_stride, const void* up, int64_t up_stride, int64_t rows, int K, int dtype, void* q,
                         float* scale, const char* what, void* stream) {
  if (dtype < 0 || dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || K < 1 || K > 0x7FFF0000 || x_stride < 0 || up_stride < 0) return fail(MOE_ERR_ARG, "%s: bad shape rows=%lld K=%d", what, (long long)rows, K);
  if (rows == 0) return MOE_OK;
  const int64_t per_row = ceil_div64(K, G);
  if (rows > 0x7FFF0000ll / per_row) return fail(MOE_ERR_UNSUPPORTED, "%s: too many groups", what);
  if (!x || (SWIGLU && !up) || !q || !scale) return fail(MOE_ERR_ARG, "%s: null pointer", what);
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  const int w = dtype == MOE_DTYPE_F32 ? 4 : 2;
  const RowParams p{x, up, x_stride, up_stride, (uint32_t)(rows * per_row), K, FastDiv((uint32_t)per_row), reinterpret_cast<uint8_t*>(q), scale};
  uintptr_t all = reinterpret_cast<uintptr_t>(x) | (uintptr_t)(x_stride * w) | (uintptr_t)((int64_t)K * w);
  if (SWIGLU) all |= reinterpret_cast<uintptr_t>(up) | (uintptr_t)(up_stride * w);
  int V = vec_bytes(all);
  if (V < w) return fail(MOE_ERR_ARG, "%s: rows are not aligned to their element type", what);
  // a vector of V bytes leaves as V / w bytes: the packed 8-bit rows are aligned for it where the base is
  if (reinterpret_cast<uintptr_t>(q) & (uintptr_t)(V / w - 1)) V = w;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MOE_DTYPE_F32) V == 16 ? launch_rows<float, 16, SWIGLU>(p, st) : launch_rows<float, 4, SWIGLU>(p, st);
#define MOE_ROWS16(T_)                                                                                             \
  V == 16 ? launch_rows<T_, 16, SWIGLU>(p, st)                                                       \
          : V >= 4 ? launch_rows<T_, 4, SWIGLU>(p, st) : launch_rows<T_, 2, SWIGLU>(p, st)
  else if (dtype == MOE_DTYPE_F16) MOE_ROWS16(__half);
  else MOE_ROWS16(__nv_bfloat16);
#undef MOE_ROWS16
  MOE_CHECK_LAUNCH(what);
  return MOE_OK;
}

}  // namespace fp8
}  // namespace moe

// ====================================================================================
extern "C" int moe_fp8_quantize_rows(const void* x, int64_t x_stride, int64_t rows, int K, int dtype, void* q, float* scale,
                                     void* stream) {
  using namespace moe::fp8;
  return quantize_rows<false>(x, x_stride, nullptr, 0, rows, K, dtype, q, scale, "fp8_quantize_rows", stream);
}

extern "C" int moe_fp8_silu_mul(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, int64_t rows, int I, int dtype,
                                void* q, float* scale, void* stream) {
  using namespace moe::fp8;
  return quantize_rows<true>(gate, gate_stride, up, up_stride, rows, I, dtype, q, scale, "fp8_silu_mul", stream);
}

extern "C" int moe_fp8_quantize_blocks(const void* w, int64_t E, int64_t rows, int K, int dtype, void* q, float* scale, void* stream) {
  using namespace moe;
  using namespace moe::fp8;
  if (dtype < 0 || dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "fp8_quantize_blocks: unknown dtype %d", dtype);
  if (E < 0 || rows < 1 || K < 1 || K > 0x7FFF0000) return fail(MOE_ERR_ARG, "fp8_quantize_blocks: bad shape %lld x %lld x %d", (long long)E, (long long)rows, K);
  if (E == 0) return MOE_OK;
  if (!w || !q || !scale) return fail(MOE_ERR_ARG, "fp8_quantize_blocks: null pointer");
  const int64_t rb = ceil_div64(rows, G), cb = ceil_div64(K, G);
  if (rb > 0x7FFFFFFFll / cb || E > 0x7FFFFFFFll / (rb * cb)) return fail(MOE_ERR_UNSUPPORTED, "fp8_quantize_blocks: too many blocks");
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  const int es = dtype == MOE_DTYPE_F32 ? 4 : 2;
  int V = vec_bytes(reinterpret_cast<uintptr_t>(w) | (uintptr_t)((int64_t)K * es));
  if (V < es) return fail(MOE_ERR_ARG, "fp8_quantize_blocks: values are not aligned to their type");
  if (V < 16 || (reinterpret_cast<uintptr_t>(q) & (uintptr_t)(16 / es - 1))) V = es;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)(E * rb * cb);
  uint8_t* o = reinterpret_cast<uint8_t*>(q);
#define MOE_BLOCKS(T_, V_) quantize_blocks_kernel<T_, V_><<<grid, 256, 0, st>>>(reinterpret_cast<const T_*>(w), rows, K, (int)rb, (int)cb, o, scale)
  if (dtype == MOE_DTYPE_F32) { if (V == 16) MOE_BLOCKS(float, 16); else MOE_BLOCKS(float, 4); }
  else if (dtype == MOE_DTYPE_F16) { if (V == 16) MOE_BLOCKS(__half, 16); else MOE_BLOCKS(__half, 2); }
  else { if (V == 16) MOE_BLOCKS(__nv_bfloat16, 16); else MOE_BLOCKS(__nv_bfloat16, 2); }
#undef MOE_BLOCKS
  MOE_CHECK_LAUNCH("quantize_blocks_kernel");
  return MOE_OK;
}
