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
#include "common.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace moe {
namespace fp8 {

constexpr int G = 128;               // elements that share a scale along a row
constexpr float TOP = 448.0f;
constexpr uint32_t TINY_BITS = 0x0D800000u;   // 2^-100: 448 / top and top / 448 stay normal numbers

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T, int V>
struct alignas(V) Pack {
  static constexpr int N = V / (int)sizeof(T);
  T e[N];
};
template <int N> struct Bytes;
template <> struct Bytes<1> { using type = uint8_t; };
template <> struct Bytes<2> { using type = uint16_t; };
template <> struct Bytes<4> { using type = uint32_t; };
template <> struct Bytes<8> { using type = uint2; };

// two fp32 -> two e4m3 in 16 bits, the first in the lower byte
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
template <int N>
__device__ __forceinline__ typename Bytes<N>::type quantize(const float* x, float inv) {
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
// |x| as bits: ordered like the magnitudes, every NaN above infinity
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

struct RowParams {
  const void* x;         // or the gate
  const void* up;
  int64_t x_stride, up_stride;   // elements
  int64_t groups;        // rows x groups of a row
  int K, per_row;        // elements and groups of a row
  uint8_t* q;
  float* scale;
};

// L lanes hold a group, I vectors of N elements each; a warp takes 32 / L groups at a time, U of them in flight per lane.
// Groups are numbered through all rows, so that short rows fill a warp too.
template <class T, int V, bool SWIGLU>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const RowParams p) {
  using P = Pack<T, V>;
  constexpr int N = P::N, L = G / N < 32 ? G / N : 32, I = G / (N * L), PER_WARP = 32 / L;
  constexpr int U = I > 1 ? 1 : (SWIGLU ? 2 : 4);
  const int lane = threadIdx.x & 31, in = lane % L;
  const int64_t warps = (int64_t)gridDim.x * 8;
  for (int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * (U * PER_WARP); first < p.groups; first += warps * (U * PER_WARP)) {
    P a[U][I], b[U][I];
    int64_t row[U];
    int col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t g = first + u * PER_WARP + lane / L;
      row[u] = g / p.per_row;
      col[u] = g < p.groups ? (int)(g - row[u] * p.per_row) * G + in * N : p.K;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int c = col[u] + i * L * N;
        if (c < p.K) {
          a[u][i] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.x) + row[u] * p.x_stride + c);
          if (SWIGLU) b[u][i] = *reinterpret_cast<const P*>(reinterpret_cast<const T*>(p.up) + row[u] * p.up_stride + c);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[I][N];
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const bool has = col[u] + i * L * N < p.K;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          x[i][j] = SWIGLU ? silu_mul(to_f32(a[u][i].e[j]), to_f32(b[u][i].e[j])) : to_f32(a[u][i].e[j]);
          m = max(m, has ? magnitude(x[i][j]) : 0u);
        }
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      const float top = __uint_as_float(max(m, TINY_BITS));
      const float inv = TOP / top;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int c = col[u] + i * L * N;
        if (c < p.K) *reinterpret_cast<typename Bytes<N>::type*>(p.q + row[u] * p.K + c) = quantize<N>(x[i], inv);
      }
      const int64_t g = first + u * PER_WARP + lane / L;
      if (in == 0 && g < p.groups) p.scale[g] = top / TOP;
    }
  }
}

// One CTA of 256 threads per 128 x 128 block, its values in registers from the one read on.  In a narrow form (V below 16
// bytes, rows of odd widths) a thread holds one element of a half row at a time: same registers, narrower accesses.
template <class T, int V>
__global__ void __launch_bounds__(256)
quantize_blocks_kernel(const T* __restrict__ w, int64_t rows, int K, int row_blocks, int col_blocks, uint8_t* __restrict__ q,
                       float* __restrict__ scale) {
  using P = Pack<T, V>;
  constexpr int N = P::N, COLS = G / N, STEP = 256 / COLS, I = G / STEP;    // vectors per row, rows at a time, vectors per thread
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
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (r0 + i * STEP < left && col < K) {
#pragma unroll
      for (int j = 0; j < N; ++j) m = max(m, magnitude(to_f32(v[i].e[j])));
    }
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, part[i]);
  const float top = __uint_as_float(max(m, TINY_BITS));
  const float inv = TOP / top;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int r = r0 + i * STEP;
    if (r < left && col < K) {
      float x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = to_f32(v[i].e[j]);
      *reinterpret_cast<typename Bytes<N>::type*>(q + base + (int64_t)r * K) = quantize<N>(x, inv);
    }
  }
  if (threadIdx.x == 0) scale[blk] = top / TOP;
}

static int vec_bytes(uintptr_t all) {
  int v = 16;
  while (v > 1 && (all & (uintptr_t)(v - 1))) v >>= 1;
  return v;
}

template <class T, int V, bool SWIGLU>
static void launch_rows(const RowParams& p, int sms, cudaStream_t st) {
  constexpr int N = V / (int)sizeof(T), L = G / N < 32 ? G / N : 32, U = G / (N * L) > 1 ? 1 : (SWIGLU ? 2 : 4);
  int64_t grid = ceil_div64(p.groups, 8 * U * (32 / L));
  if (grid > (int64_t)sms * 8) grid = (int64_t)sms * 8;
  quantize_rows_kernel<T, V, SWIGLU><<<(unsigned)grid, 256, 0, st>>>(p);
}

template <bool SWIGLU>
static int quantize_rows(const RowParams& p, int64_t rows, int dtype, const char* what, void* stream) {
  if (dtype < 0 || dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || p.K < 1 || p.x_stride < 0 || p.up_stride < 0) return fail(MOE_ERR_ARG, "%s: bad shape rows=%lld K=%d", what, (long long)rows, p.K);
  if (rows == 0) return MOE_OK;
  if (!p.x || (SWIGLU && !p.up) || !p.q || !p.scale) return fail(MOE_ERR_ARG, "%s: null pointer", what);
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  const int w = dtype == MOE_DTYPE_F32 ? 4 : 2;
  uintptr_t all = reinterpret_cast<uintptr_t>(p.x) | (uintptr_t)(p.x_stride * w) | (uintptr_t)((int64_t)p.K * w);
  if (SWIGLU) all |= reinterpret_cast<uintptr_t>(p.up) | (uintptr_t)(p.up_stride * w);
  int V = vec_bytes(all);
  if (V < w) return fail(MOE_ERR_ARG, "%s: rows are not aligned to their element type", what);
  // a vector of V bytes leaves as V / w bytes: the packed 8-bit rows are aligned for it where the base is
  if (reinterpret_cast<uintptr_t>(p.q) & (uintptr_t)(V / w - 1)) V = w;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MOE_DTYPE_F32) V == 16 ? launch_rows<float, 16, SWIGLU>(p, dev.sm_count, st) : launch_rows<float, 4, SWIGLU>(p, dev.sm_count, st);
#define MOE_ROWS16(T_)                                                                                             \
  V == 16 ? launch_rows<T_, 16, SWIGLU>(p, dev.sm_count, st)                                                       \
          : V >= 4 ? launch_rows<T_, 4, SWIGLU>(p, dev.sm_count, st) : launch_rows<T_, 2, SWIGLU>(p, dev.sm_count, st)
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
  const int per_row = K > 0 ? (K + G - 1) / G : 0;
  const RowParams p{x, nullptr, x_stride, 0, rows * per_row, K, per_row, reinterpret_cast<uint8_t*>(q), scale};
  return quantize_rows<false>(p, rows, dtype, "fp8_quantize_rows", stream);
}

extern "C" int moe_fp8_silu_mul(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, int64_t rows, int I, int dtype,
                                void* q, float* scale, void* stream) {
  using namespace moe::fp8;
  const int per_row = I > 0 ? (I + G - 1) / G : 0;
  const RowParams p{gate, up, gate_stride, up_stride, rows * per_row, I, per_row, reinterpret_cast<uint8_t*>(q), scale};
  return quantize_rows<true>(p, rows, dtype, "fp8_silu_mul", stream);
}

extern "C" int moe_fp8_quantize_blocks(const void* w, int64_t E, int64_t rows, int K, int dtype, void* q, float* scale, void* stream) {
  using namespace moe;
  using namespace moe::fp8;
  if (dtype < 0 || dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "fp8_quantize_blocks: unknown dtype %d", dtype);
  if (E < 0 || rows < 1 || K < 1) return fail(MOE_ERR_ARG, "fp8_quantize_blocks: bad shape %lld x %lld x %d", (long long)E, (long long)rows, K);
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
