// Tokens sorted by expert and back, with weights applied, and the gradients of both.
//
//   sort       the n = T*k entries (token t, slot j) by expert, stably, entries without an expert behind all others
//   permute    rows[row_of[t,j], :] = x[t, :]                               zeros in the rows behind offsets[E]
//   unpermute  y[t, :] = sum_j w[t,j] * rows[row_of[t,j], :]                entries without an expert add nothing
//
// The gradient of permute is unpermute without weights and the other way round; with weights unpermute has
//   g_rows[row_of[t,j], :] = w[t,j] * gy[t, :]        g_w[t,j] = <rows[row_of[t,j], :], gy[t, :]>
//
// All of it is bound by memory.  Every kernel goes by tokens, not by sorted rows: a token's row is read once and written to
// its k places (permute; the gradient of unpermute reads it once for every four of them), or its k rows are read and leave as
// one (unpermute), so no row is read for every copy of it and no sum needs an atomic; the order of every sum is fixed.
#include "vec.cuh"

namespace moe {
namespace perm {

// rows that hold an entry: what lies behind them is read by nobody and holds zeros
__device__ __forceinline__ int32_t live_rows(const int32_t* live, int64_t n) {
  const int32_t v = *live;
  return v < 0 ? 0 : ((int64_t)v > n ? (int32_t)n : v);
}

// One warp per token and segment of 32 * U vectors: the segment stays in registers while the k places are written.  U
// independent loads per lane, then k * U independent stores.  As many CTAs as there is work for: 8192 tokens of 7168, k = 8, bf16 172
// us, 95 % of the copy rate (185 with the CTAs that fit at a time walking over all of it).
template <int V> constexpr int permute_unroll() { return V >= 8 ? 4 : 8; }
template <int V>
__global__ void __launch_bounds__(256)
permute_kernel(const unsigned char* __restrict__ src, int64_t src_stride, const int32_t* __restrict__ row_of,
               const int32_t* __restrict__ live, int64_t T, int k, int vecs, int segs, unsigned char* __restrict__ dst) {
  using Vec = Raw<V>;
  constexpr int U = permute_unroll<V>();
  const int lane = threadIdx.x & 31;
  const int64_t n = T * k, items = T * segs, nwarps = (int64_t)gridDim.x * 8;
  const int32_t n_live = live_rows(live, n);
  for (int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); item < items; item += nwarps) {
    const int64_t t = item / segs;
    const int v0 = (int)(item - t * segs) * (32 * U) + lane;
    const Vec* s = reinterpret_cast<const Vec*>(src + t * src_stride);
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + 32 * u < vecs) v[u] = s[v0 + 32 * u];
    for (int j0 = 0; j0 < k; j0 += 32) {
      const int32_t mine = j0 + lane < k ? row_of[t * k + j0 + lane] : -1;
      const int m = min(32, k - j0);
      for (int j = 0; j < m; ++j) {
        const int32_t r = __shfl_sync(0xFFFFFFFFu, mine, j);
        if (r < 0 || r >= n) continue;
        Vec* d = reinterpret_cast<Vec*>(dst) + (int64_t)r * vecs;
        const bool has = r < n_live;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (v0 + 32 * u < vecs) d[v0 + 32 * u] = has ? v[u] : Vec{};
      }
    }
  }
}

// One CTA per token: its rows' numbers and weights stay in registers (k <= J, ONE) while the threads walk over the width.
// The J rows' pieces are in flight before the first is added, U of them each where vectors are narrow; they are added in
// slot order, in fp32, with one rounding at the end.  65536 rows of 7168, k = 8, bf16: 161 us, the copy rate (a warp per token and
// piece of the width looked up its rows for every piece: 272 us); 32768 fp32 rows of 2048, k = 4: 54 us, 60 with J = 8.
template <class T, int V, bool ONE, int J>
__global__ void __launch_bounds__(256)
unpermute_kernel(const T* __restrict__ rows, int64_t rows_stride, const int32_t* __restrict__ row_of,
                 const int32_t* __restrict__ live, const float* __restrict__ weights, int64_t tokens, int k, int vecs,
                 T* __restrict__ out) {
  using P = Raw<V>;
  constexpr int N = V / (int)sizeof(T), U = V == 16 ? 1 : (V == 8 ? 2 : 4);
  const int32_t n_live = live_rows(live, tokens * k);
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    int32_t r[J];
    float w[J];
    auto look_up = [&](int j0) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        r[j] = -1;
        w[j] = 1.f;
        if (j0 + j < k) {
          r[j] = row_of[t * k + j0 + j];
          if (weights) w[j] = weights[t * k + j0 + j];
          if (r[j] >= n_live) r[j] = -1;
        }
      }
    };
    if (ONE) look_up(0);
    P* d = reinterpret_cast<P*>(out) + t * vecs;
    for (int v0 = threadIdx.x; v0 < vecs; v0 += blockDim.x * U) {
      float acc[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[u][i] = 0.f;
      for (int j0 = 0; j0 < (ONE ? 1 : k); j0 += J) {
        if (!ONE) look_up(j0);
        P p[J][U];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const P* s = reinterpret_cast<const P*>(rows + (int64_t)r[j] * rows_stride);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (r[j] >= 0 && v0 + u * (int)blockDim.x < vecs) p[j][u] = s[v0 + u * blockDim.x];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (r[j] < 0) continue;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float x[N];
            unpack<T, V>(p[j][u], x);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[u][i] = fmaf(w[j], x[i], acc[u][i]);      // by 1 where there are no weights: the sum itself
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * (int)blockDim.x < vecs) d[v0 + u * blockDim.x] = pack<T, V>(acc[u]);
    }
  }
}

// One CTA per token and run of up to four slots: a piece of gy is read once, multiplied into the rows' places and into as many
// sums over the width, which the CTA adds up at the end: lanes by shuffles, warps in their order.  Eight slots at a time read
// gy once less, but keep 128 registers a thread (65536 rows of 7168, k = 8: 330 us against 310).
constexpr int GRAD_SLOTS = 4;
template <class T, int V>
__global__ void __launch_bounds__(256)
unpermute_grad_kernel(const T* __restrict__ gy, int64_t gy_stride, const T* __restrict__ rows, int64_t rows_stride,
                      const int32_t* __restrict__ row_of, const int32_t* __restrict__ live, const float* __restrict__ weights,
                      int64_t tokens, int k, int vecs, T* __restrict__ g_rows, float* __restrict__ g_w) {
  using P = Raw<V>;
  constexpr int N = V / (int)sizeof(T), J = GRAD_SLOTS, U = V == 16 ? 1 : (V == 8 ? 2 : 4);
  __shared__ float part[8][J];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const int runs = (k + J - 1) / J;
  const int64_t n = tokens * k;
  const int32_t n_live = live_rows(live, n);
  for (int64_t item = blockIdx.x; item < tokens * runs; item += gridDim.x) {
    const int64_t t = item / runs;
    const int j0 = (int)(item - t * runs) * J, m = min(J, k - j0);
    int32_t r[J];
    float w[J], dot[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      r[j] = j < m ? row_of[t * k + j0 + j] : -1;
      if (r[j] >= n) r[j] = -1;
      w[j] = j < m ? weights[t * k + j0 + j] : 0.f;
      dot[j] = 0.f;
    }
    const P* g = reinterpret_cast<const P*>(gy + t * gy_stride);
    for (int v0 = threadIdx.x; v0 < vecs; v0 += blockDim.x * U) {
      P graw[U], p[J][U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * (int)blockDim.x < vecs) graw[u] = g[v0 + u * blockDim.x];
      if (g_w) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const P* s = reinterpret_cast<const P*>(rows + (int64_t)r[j] * rows_stride);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (r[j] >= 0 && r[j] < n_live && v0 + u * (int)blockDim.x < vecs) p[j][u] = s[v0 + u * blockDim.x];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = v0 + u * blockDim.x;
        if (v >= vecs) break;
        float gf[N];
        unpack<T, V>(graw[u], gf);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (r[j] < 0) continue;
          const bool has = r[j] < n_live;
          if (g_w && has) {
            float x[N];
            unpack<T, V>(p[j][u], x);
#pragma unroll
            for (int i = 0; i < N; ++i) dot[j] = fmaf(x[i], gf[i], dot[j]);
          }
          if (g_rows) {
            float o[N];
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = has ? w[j] * gf[i] : 0.f;
            reinterpret_cast<P*>(g_rows)[(int64_t)r[j] * vecs + v] = pack<T, V>(o);
          }
        }
      }
    }
    if (g_w) {
#pragma unroll
      for (int j = 0; j < J; ++j) dot[j] = warp_sum(dot[j]);
      if (lane == 0) {
#pragma unroll
        for (int j = 0; j < J; ++j) part[warp][j] = dot[j];
      }
      __syncthreads();
      if (threadIdx.x < m) {
        float s = 0.f;
        for (int q = 0; q < nwarps; ++q) s += part[q][threadIdx.x];
        g_w[t * k + j0 + threadIdx.x] = s;
      }
      __syncthreads();
    }
  }
}

// threads of a CTA that walks over `vecs` vectors of V bytes
static unsigned threads_for(int vecs, int V) {
  const int work = (vecs + (V == 16 ? 0 : (V == 8 ? 1 : 3))) / (V == 16 ? 1 : (V == 8 ? 2 : 4));
  return work >= 256 ? 256u : (unsigned)((work + 31) / 32 * 32);
}

static int elem_bytes(int dtype) { return dtype == MOE_DTYPE_F32 ? 4 : 2; }

static unsigned grid_for(int64_t items, int64_t per_cta, int64_t cap) {
  int64_t b = ceil_div64(items, per_cta);
  return (unsigned)(b < 1 ? 1 : (b > cap ? cap : b));
}

// CTAs that an SM can hold, for kernels that walk over the tokens: rows of few vectors make small ones
static int64_t resident(int sms, unsigned threads) { return (int64_t)sms * (threads >= 64 ? 2048 / threads : 32); }

}  // namespace perm
}  // namespace moe

// ====================================================================================
// one group more than experts; no number of them that the histogram takes is anywhere near the largest int
constexpr int SORT_MAX_E = 1 << 30;
extern "C" size_t moe_sort_workspace(int64_t n, int E) { return E < 1 || E > SORT_MAX_E ? 0 : moe_route_histogram_workspace(n, E + 1); }

extern "C" int moe_sort(const void* ids, int idx_is_int64, int64_t n, int E, int32_t* counts, int32_t* offsets, int32_t* perm,
                        int32_t* row_of, void* ws, size_t ws_bytes, void* stream) {
  using namespace moe;
  if (E < 1) return fail(MOE_ERR_ARG, "sort: bad expert count %d", E);
  if (E > SORT_MAX_E) return fail(MOE_ERR_UNSUPPORTED, "sort: E=%d too large", E);
  if (n > 0 && (!perm || !row_of)) return fail(MOE_ERR_ARG, "sort: null perm/row_of");
  return route_histogram_ex(ids, idx_is_int64, n, E + 1, nullptr, counts, offsets, perm, row_of, ws, ws_bytes, nullptr, stream,
                            ROUTE_KEEP_ALL, false);
}

extern "C" int moe_permute(const void* src, int64_t src_stride, int64_t row_bytes, const int32_t* row_of, const int32_t* live,
                           int64_t T, int k, void* dst, void* stream) {
  using namespace moe;
  using namespace moe::perm;
  if (T < 0 || k < 1 || row_bytes < 1 || src_stride < 0) return fail(MOE_ERR_ARG, "permute: bad shape T=%lld k=%d row bytes=%lld stride=%lld", (long long)T, k, (long long)row_bytes, (long long)src_stride);
  if (T == 0) return MOE_OK;
  if (!src || !row_of || !live || !dst) return fail(MOE_ERR_ARG, "permute: null pointer");
  if (T > 0x7FFFFFFFll || T * k > 0x7FFFFFFFll || row_bytes > 0x7FFF0000ll) return fail(MOE_ERR_UNSUPPORTED, "permute: too many rows or too wide ones");
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  const int V = vec_bytes(reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | (uintptr_t)src_stride | (uintptr_t)row_bytes);
  const int vecs = (int)(row_bytes / V), segs = (vecs + (V >= 8 ? 127 : 255)) / (V >= 8 ? 128 : 256);
  const unsigned grid = grid_for(T * segs, 8, 0x7FFFFFFFll);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const unsigned char* s = reinterpret_cast<const unsigned char*>(src);
  unsigned char* d = reinterpret_cast<unsigned char*>(dst);
#define MOE_PERMUTE(V_) permute_kernel<V_><<<grid, 256, 0, st>>>(s, src_stride, row_of, live, T, k, vecs, segs, d)
  switch (V) {
    case 16: MOE_PERMUTE(16); break;
    case 8: MOE_PERMUTE(8); break;
    case 4: MOE_PERMUTE(4); break;
    case 2: MOE_PERMUTE(2); break;
    default: MOE_PERMUTE(1); break;
  }
#undef MOE_PERMUTE
  MOE_CHECK_LAUNCH("permute_kernel");
  return MOE_OK;
}

template <class T, int V>
static void launch_unpermute(const void* rows, int64_t stride, const int32_t* row_of, const int32_t* live, const float* w, int64_t tokens,
                             int k, int64_t H, void* out, int sms, cudaStream_t st) {
  using namespace moe::perm;
  const int vecs = (int)(H * sizeof(T) / V);
  const unsigned threads = threads_for(vecs, V), grid = grid_for(tokens, 1, resident(sms, threads));
  const T* r = reinterpret_cast<const T*>(rows);
  T* o = reinterpret_cast<T*>(out);
  if (k <= 4) unpermute_kernel<T, V, true, 4><<<grid, threads, 0, st>>>(r, stride, row_of, live, w, tokens, k, vecs, o);
  else if (k <= 8) unpermute_kernel<T, V, true, 8><<<grid, threads, 0, st>>>(r, stride, row_of, live, w, tokens, k, vecs, o);
  else unpermute_kernel<T, V, false, 8><<<grid, threads, 0, st>>>(r, stride, row_of, live, w, tokens, k, vecs, o);
}

extern "C" int moe_unpermute(const void* rows, int64_t rows_stride, const int32_t* row_of, const int32_t* live, const float* weights,
                             int64_t T, int k, int64_t H, int dtype, void* out, void* stream) {
  using namespace moe;
  using namespace moe::perm;
  if (dtype < 0 || dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "unpermute: unknown dtype %d", dtype);
  if (T < 0 || k < 1 || H < 1 || rows_stride < 0) return fail(MOE_ERR_ARG, "unpermute: bad shape T=%lld k=%d H=%lld", (long long)T, k, (long long)H);
  if (T == 0) return MOE_OK;
  if (!rows || !row_of || !live || !out) return fail(MOE_ERR_ARG, "unpermute: null pointer");
  if (T > 0x7FFFFFFFll || T * k > 0x7FFFFFFFll || H > 0x1FFF0000ll) return fail(MOE_ERR_UNSUPPORTED, "unpermute: too many rows or too wide ones");
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  const int w = elem_bytes(dtype);
  const int V = vec_bytes(reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(out) | (uintptr_t)(rows_stride * w) | (uintptr_t)(H * w));
  if (V < w) return fail(MOE_ERR_ARG, "unpermute: rows are not aligned to their element type");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define MOE_UNPERMUTE(T_, V_) launch_unpermute<T_, V_>(rows, rows_stride, row_of, live, weights, T, k, H, out, dev.sm_count, st)
#define MOE_UNPERMUTE16(T_) (V == 16 ? MOE_UNPERMUTE(T_, 16) : V == 8 ? MOE_UNPERMUTE(T_, 8) : V == 4 ? MOE_UNPERMUTE(T_, 4) : MOE_UNPERMUTE(T_, 2))
  if (dtype == MOE_DTYPE_F32) V == 16 ? MOE_UNPERMUTE(float, 16) : V == 8 ? MOE_UNPERMUTE(float, 8) : MOE_UNPERMUTE(float, 4);
  else if (dtype == MOE_DTYPE_F16) MOE_UNPERMUTE16(__half);
  else MOE_UNPERMUTE16(__nv_bfloat16);
#undef MOE_UNPERMUTE16
#undef MOE_UNPERMUTE
  MOE_CHECK_LAUNCH("unpermute_kernel");
  return MOE_OK;
}

template <class T, int V>
static void launch_unpermute_grad(const void* gy, int64_t gy_stride, const void* rows, int64_t rows_stride, const int32_t* row_of,
                                  const int32_t* live, const float* w, int64_t tokens, int k, int64_t H, void* g_rows, float* g_w,
                                  int sms, cudaStream_t st) {
  using namespace moe::perm;
  const int vecs = (int)(H * sizeof(T) / V);
  const unsigned threads = threads_for(vecs, V);
  const T *g = reinterpret_cast<const T*>(gy), *r = reinterpret_cast<const T*>(rows);
  T* gr = reinterpret_cast<T*>(g_rows);
  const int64_t items = tokens * ((k + GRAD_SLOTS - 1) / GRAD_SLOTS);
  unpermute_grad_kernel<T, V><<<grid_for(items, 1, resident(sms, threads)), threads, 0, st>>>(g, gy_stride, r, rows_stride, row_of, live, w, tokens, k,
                                                                                     vecs, gr, g_w);
}

extern "C" int moe_unpermute_grad(const void* gy, int64_t gy_stride, const void* rows, int64_t rows_stride, const int32_t* row_of,
                                  const int32_t* live, const float* weights, int64_t T, int k, int64_t H, int dtype, void* g_rows,
                                  float* g_w, void* stream) {
  using namespace moe;
  using namespace moe::perm;
  if (dtype < 0 || dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "unpermute_grad: unknown dtype %d", dtype);
  if (T < 0 || k < 1 || H < 1 || gy_stride < 0 || rows_stride < 0) return fail(MOE_ERR_ARG, "unpermute_grad: bad shape T=%lld k=%d H=%lld", (long long)T, k, (long long)H);
  if (T == 0 || (!g_rows && !g_w)) return MOE_OK;
  if (!gy || !row_of || !live || !weights || (g_w && !rows)) return fail(MOE_ERR_ARG, "unpermute_grad: null pointer");
  if (T > 0x7FFFFFFFll || T * k > 0x7FFFFFFFll || H > 0x1FFF0000ll) return fail(MOE_ERR_UNSUPPORTED, "unpermute_grad: too many rows or too wide ones");
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  const int w = elem_bytes(dtype);
  uintptr_t all = reinterpret_cast<uintptr_t>(gy) | (uintptr_t)(gy_stride * w) | (uintptr_t)(H * w) | reinterpret_cast<uintptr_t>(g_rows);
  if (g_w) all |= reinterpret_cast<uintptr_t>(rows) | (uintptr_t)(rows_stride * w);
  const int V = vec_bytes(all);
  if (V < w) return fail(MOE_ERR_ARG, "unpermute_grad: rows are not aligned to their element type");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define MOE_UNPERMUTE(T_, V_) \
  launch_unpermute_grad<T_, V_>(gy, gy_stride, rows, rows_stride, row_of, live, weights, T, k, H, g_rows, g_w, dev.sm_count, st)
#define MOE_UNPERMUTE16(T_) (V == 16 ? MOE_UNPERMUTE(T_, 16) : V == 8 ? MOE_UNPERMUTE(T_, 8) : V == 4 ? MOE_UNPERMUTE(T_, 4) : MOE_UNPERMUTE(T_, 2))
  if (dtype == MOE_DTYPE_F32) V == 16 ? MOE_UNPERMUTE(float, 16) : V == 8 ? MOE_UNPERMUTE(float, 8) : MOE_UNPERMUTE(float, 4);
  else if (dtype == MOE_DTYPE_F16) MOE_UNPERMUTE16(__half);
  else MOE_UNPERMUTE16(__nv_bfloat16);
#undef MOE_UNPERMUTE16
#undef MOE_UNPERMUTE
  MOE_CHECK_LAUNCH("unpermute_grad_kernel");
  return MOE_OK;
}
