// 8-bit GEMM with a scale for each block of 128, dense or grouped by expert, for sm_100a.
//
//   Y[m, n] = sum over kb of  sa[m, kb] * sb[n / 128, kb] * ( sum over the 128 k of block kb of  A[m, k] * B[n, k] )
//
// A [rows, K] and B [E, N, K] are e4m3, the inner sums are taken by tcgen05.mma (kind::f8f6f4, fp32 accumulators in tensor
// memory), and because the scales change every 128 k, each block's sum leaves tensor memory and is added, scaled, to fp32
// accumulators in registers:
//
//   warp 0      TMA producer: per k-block one A box (128 rows x 128 bytes, 32 for a tile of few rows) and one B box (BN rows),
//               128-byte swizzle, into a ring of shared-memory stages;
//   warp 1      MMA issuer: four instructions (K = 32) per k-block into one of two accumulators in tensor memory, in turn;
//   warps 2..9  one tile row and half of the tile's columns per thread: acc += (sa * sb) * block sum, while the other
//               accumulator is being filled; after the last block convert and store.
//
// What bounds it.  Many rows: a k-block of a 128 x 256 tile takes about 940 clocks, of which the tensor cores need 512 (8192 x 4096 x
// 7168, clock64 around the 392 k-blocks of a CTA; from idle and back to back alike).  With the additions left out it takes 700, with
// the loads from tensor memory left out as well 690: the operands come that slowly with nothing beside them, and the additions cost
// the rest.  An accumulating warp by itself needs about 500.  The power cap makes every clock longer: 232 to 245 us from idle, 277
// back to back at 985 W and 1.46 GHz (2.07 to 1.74 PFLOP/s); the library's product without block scales 178 and 198.  A form on CTA
// pairs (cta_group::2, two thirds of the operand traffic per SM) ran at 512 clocks a k-block without the additions, but with them was
// no faster: 265 to 288 us back to back where this one took 269, 160 to 172 against 162 at 8192 x 7168 x 2048, 667 to 725 against 650 on 64
// experts.  Sixteen accumulating warps instead of eight: 307 against 258.
// Few rows: reading the weights: 250 rows on 111 experts of 2048 x 4096 in 166 us, 5.6 TB/s.
//
// K need not be a multiple of 128: TMA fills what lies behind it with zeros.  Rows of a tile behind its group are computed
// and not stored.  Every barrier wait is bounded in time, as in the 16-bit kernels.
#include "sm100.cuh"

#include <cuda_fp16.h>

namespace moe {
namespace gemm8 {

using namespace moe::gemm;

constexpr int BM = 128;
constexpr int BK = 128;                // bytes = elements: one swizzle row, one scale block
constexpr int UMMA_K = 32;
constexpr int NUM_THREADS = 320;
constexpr int EPI_WARPS = 8;
constexpr int MAX_E = 1024;
constexpr int FEW_ROWS = 32;            // tiles of at most so many rows bring no more of A

constexpr int STAGING_PITCH = 17;       // floats: 16 columns and one, so that rows and columns are free of bank conflicts
constexpr int MAX_SPLIT = 8;            // CTAs of a cluster that share a tile's k-blocks

// AR: rows of A that a stage has room for: a tile's 128, or FEW_ROWS where no tile can have more.  The instructions read 128
// rows all the same, those behind the room from whatever follows in the stage, and nothing of what they make of it is stored.
template <int BN, int AR>
struct Cfg {
  static constexpr int A_BYTES = AR * BK;
  static constexpr int B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static_assert(STAGE_BYTES >= BM * BK, "an instruction stays inside its stage");
  static constexpr int STAGES = (192 * 1024) / STAGE_BYTES;     // BN = 256: 4, 128: 6, with 32 rows of A 9
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int BAR_OFFSET = STAGES * STAGE_BYTES;
  static constexpr int SLOT_OFFSET = BAR_OFFSET + (2 * STAGES + 5) * 8;
  static constexpr int TABLE_OFFSET = (SLOT_OFFSET + 16 + 15) & ~15;
  static constexpr int STAGING_OFFSET = (TABLE_OFFSET + 2 * (MAX_E + 1) * 4 + 15) & ~15;   // rows of Y that take no vectors
  static constexpr int SMEM_BYTES = STAGING_OFFSET + EPI_WARPS * 32 * STAGING_PITCH * 4 + 1024;   // + alignment slack
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
  static constexpr int PART_PITCH = BN + 4;                     // floats per row of a partial tile, which lies where the stages were
  static_assert(BM * PART_PITCH * 4 <= BAR_OFFSET, "a partial tile fits the stages");
};

struct Params {
  const float* sa;
  int64_t sa_row, sa_k;          // strides
  const float* sb;               // [E, ceil(N / 128), ceil(K / 128)]
  const int32_t* offsets;        // null: one group of all rows
  void* Y;
  int64_t ldy;
  int rows, K, N, E;
  int n_tiles, k_blocks, n_blocks;
  int out;                       // MOE_DTYPE_*
  int vec_store;                 // rows of Y take stores of 16 (1) or 32 (2) bytes
  int zero_tail;                 // rows of no group are set to zero
  int a_box_rows;                // rows of A that a stage brings (fewer than a tile's where A has fewer); FEW_ROWS for a tile of few
  int32_t* status;
};

// One lane of the warp, the same at every call: issued under its predicate in code that the whole warp runs, the instructions
// below take their operands from uniform registers.  In a branch of one thread each of them is moved there first: the four
// instructions of a k-block with their commits took 610 clocks to issue so, and 360 like this (N = 128, nothing else running;
// N = 256, which takes the tensor cores 512: 611 and 512).
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void umma_e4m3(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void umma_commit_elected(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(bar), "r"(elected)
      : "memory");
}
// D fp32 (bit 4), A and B e4m3 (formats 0), both K-major
__host__ __device__ constexpr uint32_t make_idesc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Two fp32 in one 64-bit register pair.  The scaled additions are fma.rn.f32x2: plain fma instructions take the tensor cores'
// time.  Measured, clocks for the four instructions of a k-block (128 x 256) beside accumulating warps that never wait: alone
// 518, beside fma only 1520, beside fma.rn.f32x2 only 571; with the tensor-memory loads 916 and 670.
typedef unsigned long long f32x2;
// 32 lanes x 16 consecutive fp32 columns of tensor memory, waited for, in pairs: one statement, so that no use of the values
// can be moved above the wait
__device__ __forceinline__ void tmem_ld16_pairs(uint32_t taddr, f32x2 (&r)[8]) {
  asm volatile(
      "{\n\t.reg .b32 t<16>;\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {t0, t1, t2, t3, t4, t5, t6, t7, t8, t9, t10, t11, t12, t13, t14, t15}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n\t"
      "mov.b64 %0, {t0, t1};\n\t"
      "mov.b64 %1, {t2, t3};\n\t"
      "mov.b64 %2, {t4, t5};\n\t"
      "mov.b64 %3, {t6, t7};\n\t"
      "mov.b64 %4, {t8, t9};\n\t"
      "mov.b64 %5, {t10, t11};\n\t"
      "mov.b64 %6, {t12, t13};\n\t"
      "mov.b64 %7, {t14, t15};\n\t"
      "}"
      : "=l"(r[0]), "=l"(r[1]), "=l"(r[2]), "=l"(r[3]), "=l"(r[4]), "=l"(r[5]), "=l"(r[6]), "=l"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ f32x2 pair_of(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ void fma2(f32x2& acc, f32x2 v, f32x2 s) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ bool no_normal_number(float s) { return (__float_as_uint(s) << 1) - 0x01000000u >= 0xFE000000u; }
// A block's sum times both of its scales: (sum * pre) * post.  Their product alone serves, and pre is 1, while it is a normal
// number.  Where two finite scales leave that range the sum meets the larger one first if their product is too small, the smaller
// one first if it is too large, so that what is rounded in between is no further from the result's range than the result.  A
// row's bits do not depend on which way its neighbours in the warp go: times 1 is exact.
__device__ __forceinline__ void split_scale(float a, float b, float& pre, float& post) {
  const float s = a * b, big = fmaxf(fabsf(a), fabsf(b));
  pre = 1.0f;
  post = s;
  if (!no_normal_number(s) || a == 0.0f || b == 0.0f || !(big <= 0x1.fffffep127f)) return;    // zero and infinity stay what they are
  const bool a_first = (fabsf(s) < 1.0f) == (fabsf(a) == big);
  pre = a_first ? a : b;
  post = a_first ? b : a;
}

// The wait of the accumulating warps, without the call of mbar_wait: around a call every register is spoken for.
__device__ __forceinline__ bool mbar_wait_inline(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status, int site) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t until = global_timer_ns() + WAIT_LIMIT_NS;
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (global_timer_ns() > until) break;
  }
  if (atomicExch((int*)abort_flag, 1) == 0 && status) {
    status[0] = ST_WAIT_TIMEOUT;
    status[1] = site;
    status[2] = (int32_t)blockIdx.x;
  }
  return false;
}

struct Tile {
  int e, row0, row_end, n_tile;
};
// tstart[e] = row tiles of the groups before e.  Tile ids: group, then bands of eight column tiles, then row tile, then column
// tile, so that what the SMs work on at a time is a block of the output that is neither tall nor wide, and its rows of A and
// B stay in L2 meanwhile (column tiles one after the other -> this: 8192 x 4096 x 7168 247 -> 235 us, 32768 rows on 64 experts of
// 2048 x 7168, Zipf load, 669 -> 573 us; four or sixteen tiles to a band are no better).
constexpr int BAND = 8;
__device__ __forceinline__ Tile decode_tile(int id, const int32_t* tstart, const int32_t* offs, int E, int NT) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tstart[mid + 1] * NT > id) hi = mid; else lo = mid + 1;
  }
  const int local = id - tstart[lo] * NT, mt = tstart[lo + 1] - tstart[lo];
  const int band = local / (mt * BAND), in = local - band * mt * BAND, width = min(BAND, NT - band * BAND), m = in / width;
  Tile t;
  t.e = lo;
  t.n_tile = band * BAND + in - m * width;
  t.row0 = offs[lo] + m * BM;
  t.row_end = offs[lo + 1];
  return t;
}
__device__ __forceinline__ int group_tiles(const int32_t* offs, int e) { return (offs[e + 1] - offs[e] + BM - 1) / BM; }

// One warp: offs[0 .. E] made a prefix sum of groups inside the tensor (every entry cut to [0, rows] already, none below the one
// before it), so that a table that is none leaves every access in bounds; then the row tiles before each group.
__device__ __forceinline__ void tile_prefix(int32_t* tstart, int32_t* offs, int E, int lane) {
  const int per = (E + 32) / 32;
  const int lo = min(E + 1, lane * per), hi = min(E + 1, lo + per);
  int top = 0;
  for (int i = lo; i < hi; ++i) offs[i] = top = max(top, offs[i]);
  int before = top;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, before, o);
    if (lane >= o) before = max(before, v);
  }
  before = __shfl_up_sync(0xFFFFFFFFu, before, 1);
  if (lane > 0)
    for (int i = lo; i < hi; ++i) offs[i] = max(before, offs[i]);
  __syncwarp();
  const int e_lo = min(E, lo), e_hi = min(E, hi);
  int sum = 0;
  for (int e = e_lo; e < e_hi; ++e) sum += group_tiles(offs, e);
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += v;
  }
  int run = inc - sum;
  for (int e = e_lo; e < e_hi; ++e) { tstart[e] = run; run += group_tiles(offs, e); }
  if (lane == 31) tstart[E] = inc;
}

__device__ __forceinline__ uint32_t pack16(f32x2 pair, int out) {
  const float2 v = unpair(pair);
  if (out == MOE_DTYPE_F16) { __half2 h = __floats2half2_rn(v.x, v.y); return *reinterpret_cast<uint32_t*>(&h); }
  __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint16_t one16(float a, int out) {
  return out == MOE_DTYPE_F16 ? __half_as_ushort(__float2half_rn(a)) : __bfloat16_as_ushort(__float2bfloat16_rn(a));
}

__device__ __forceinline__ f32x2 pack16x2(f32x2 a, f32x2 b, int out) {
  return (f32x2)pack16(a, out) | ((f32x2)pack16(b, out) << 32);
}
// 32 bytes at once, a whole sector: threads hold rows, so narrower stores of a warp leave half of every sector to the next one
// (8192 x 7168 x 2048, bf16 output: 183 -> 148 us)
__device__ __forceinline__ void store32(void* p, f32x2 a, f32x2 b, f32x2 c, f32x2 d) {
  asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(p), "l"(a), "l"(b), "l"(c), "l"(d) : "memory");
}

// columns [col0, col0 + COLS) of the warp's rows row .. row + 31 (one per lane), those below row_end and N, rounded to the
// output type
template <int COLS>
__device__ __forceinline__ void store_rows(const Params& p, int row0, int row_end, int lane, int col0, const f32x2 (&acc)[COLS / 2], float* staging) {
  const int out = p.out;
  const int64_t row = row0 + lane;
  if (p.vec_store) {
    if (row >= row_end) return;
    unsigned char* y = reinterpret_cast<unsigned char*>(p.Y) + (row * p.ldy + col0) * (out == MOE_DTYPE_F32 ? 4 : 2);
    if (out == MOE_DTYPE_F32 && p.vec_store == 2) {
#pragma unroll
      for (int j = 0; j < COLS / 2; j += 4)
        if (col0 + 2 * j < p.N) store32(y + j * 8, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
    } else if (out == MOE_DTYPE_F32) {
#pragma unroll
      for (int j = 0; j < COLS / 2; j += 2)
        if (col0 + 2 * j < p.N) *reinterpret_cast<ulonglong2*>(y + j * 8) = make_ulonglong2(acc[j], acc[j + 1]);
    } else if (p.vec_store == 2) {
#pragma unroll
      for (int j = 0; j < COLS / 2; j += 8)
        if (col0 + 2 * j < p.N)
          store32(y + j * 4, pack16x2(acc[j], acc[j + 1], out), pack16x2(acc[j + 2], acc[j + 3], out), pack16x2(acc[j + 4], acc[j + 5], out),
                  pack16x2(acc[j + 6], acc[j + 7], out));
    } else {
#pragma unroll
      for (int j = 0; j < COLS / 2; j += 4)
        if (col0 + 2 * j < p.N)
          *reinterpret_cast<uint4*>(y + j * 4) = make_uint4(pack16(acc[j], out), pack16(acc[j + 1], out), pack16(acc[j + 2], out), pack16(acc[j + 3], out));
    }
    return;
  }
  // rows of no alignment: 16 columns at a time through shared memory, from where half a warp writes neighbours of one row
  // (188 x 7699 x 464: 25.1 -> 9.6 us)
  const int n_rows = min(32, row_end - row0), cc = lane & 15;
#pragma unroll
  for (int c = 0; c < COLS / 16; ++c) {
    if (col0 + c * 16 >= p.N) break;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 v = unpair(acc[c * 8 + j]);
      staging[lane * STAGING_PITCH + 2 * j] = v.x;
      staging[lane * STAGING_PITCH + 2 * j + 1] = v.y;
    }
    __syncwarp();
    const int col = col0 + c * 16 + cc;
#pragma unroll 4
    for (int r = lane >> 4; r < n_rows; r += 2) {
      const float v = staging[r * STAGING_PITCH + cc];
      const int64_t at = (int64_t)(row0 + r) * p.ldy + col;
      if (col < p.N) {
        if (out == MOE_DTYPE_F32) reinterpret_cast<float*>(p.Y)[at] = v;
        else reinterpret_cast<uint16_t*>(p.Y)[at] = one16(v, out);
      }
    }
  }
}
__device__ __forceinline__ void store_four(const Params& p, int64_t row, int col, float4 v) {
  unsigned char* y = reinterpret_cast<unsigned char*>(p.Y) + (row * p.ldy + col) * (p.out == MOE_DTYPE_F32 ? 4 : 2);
  if (p.vec_store) {
    if (col >= p.N) return;                     // N is a multiple of four or eight then
    if (p.out == MOE_DTYPE_F32) *reinterpret_cast<float4*>(y) = v;
    else *reinterpret_cast<uint2*>(y) = make_uint2(pack16(pair_of(v.x, v.y), p.out), pack16(pair_of(v.z, v.w), p.out));
  } else {
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (col + j < p.N) {
        if (p.out == MOE_DTYPE_F32) reinterpret_cast<float*>(y)[j] = e[j];
        else reinterpret_cast<uint16_t*>(y)[j] = one16(e[j], p.out);
      }
    }
  }
}
// four floats of a CTA of this cluster (an address from map_to_cta)
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// rows of no group, before the first one and behind the last, set to zero; warps w of n
__device__ __forceinline__ void zero_rows(const Params& p, int64_t ahead, int64_t behind, int64_t w, int64_t n, int lane) {
  for (int64_t i = w; i < ahead + p.rows - behind; i += n) {
    const int64_t r = i < ahead ? i : behind + i - ahead;
    unsigned char* y = reinterpret_cast<unsigned char*>(p.Y) + r * p.ldy * (p.out == MOE_DTYPE_F32 ? 4 : 2);
    if (p.vec_store) {
      for (int c = lane; c < (p.out == MOE_DTYPE_F32 ? p.N / 4 : p.N / 8); c += 32) reinterpret_cast<uint4*>(y)[c] = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    for (int c = lane; c < p.N; c += 32) {
      if (p.out == MOE_DTYPE_F32) reinterpret_cast<uint32_t*>(y)[c] = 0u;
      else reinterpret_cast<uint16_t*>(y)[c] = 0;
    }
  }
}

// SPLIT: the CTAs of a cluster take a run of the k-blocks each, of one tile per cluster; what they have accumulated meets in
// shared memory and is added in the order of the CTAs.  For products of few tiles, which would leave most SMs without one.
template <int BN, bool SPLIT, int AR>
__global__ void __launch_bounds__(NUM_THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmAFew, const __grid_constant__ CUtensorMap tmB,
                const Params p) {
  using C = Cfg<BN, AR>;
  constexpr int STAGES = C::STAGES, COLS = BN / 2;       // COLS: columns of an epilogue thread
  extern __shared__ unsigned char smem_dyn[];
  // the swizzle pattern needs 1024-byte aligned stage buffers
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFFSET);
  // bars[0..S) full, [S..2S) empty, [2S..2S+2) tmem_full, [2S+2..2S+4) tmem_empty, [2S+4] drain
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::SLOT_OFFSET);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::SLOT_OFFSET + 8);
  int32_t* tstart = reinterpret_cast<int32_t*>(smem + C::TABLE_OFFSET);
  int32_t* offs = tstart + (MAX_E + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
  const uint32_t tfull0 = smem_u32(bars + 2 * STAGES), tempty0 = smem_u32(bars + 2 * STAGES + 2);
  const uint32_t drain_bar = smem_u32(bars + 2 * STAGES + 4);
  const int E = p.E, NT = p.n_tiles;
  const int S = SPLIT ? (int)cluster_nctarank() : 1, rank = SPLIT ? (int)cluster_ctarank() : 0;
  const int first_tile = SPLIT ? (int)blockIdx.x / S : (int)blockIdx.x, tile_step = SPLIT ? 1 << 30 : (int)gridDim.x;
  const int kb0 = SPLIT ? (int)((int64_t)p.k_blocks * rank / S) : 0;                      // this CTA's k-blocks
  const int kb1 = SPLIT ? (int)((int64_t)p.k_blocks * (rank + 1) / S) : p.k_blocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, EPI_WARPS); }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmAFew);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  for (int e = threadIdx.x; e <= E; e += blockDim.x) offs[e] = p.offsets ? min(max(p.offsets[e], 0), p.rows) : (e == 0 ? 0 : p.rows);
  __syncthreads();
  if (warp == 2) tile_prefix(tstart, offs, E, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int total_tiles = tstart[E] * NT;

  if (warp == 0) {
    // ===================================================================== TMA producer
    int stage = 0;
    uint32_t phase = 0, issued = 0;
    bool ok = true;
    // weights of a group with one row tile are read once and leave L2 first (1000 rows on 32 experts of 4096 x 2048, Zipf load, 55.8 ->
    // 52.7 us)
    const uint64_t pol_first = make_policy_evict_first();
    uint64_t pol_normal;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol_normal));
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      const Tile t = decode_tile(tile, tstart, offs, E, NT);
      const bool few = t.row_end - t.row0 <= FEW_ROWS;
      const uint32_t tx = (few ? FEW_ROWS : p.a_box_rows) * BK + C::B_BYTES;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, abort_flag, p.status, 31)) { ok = false; break; }
        if (lane == 0) {
          const uint32_t full = full0 + 8 * stage;
          const uint32_t sa = smem_u32(smem + stage * C::STAGE_BYTES);
          mbar_arrive_expect_tx(full, tx);
          tma_load_2d(sa, few ? &tmAFew : &tmA, full, kb * BK, t.row0);
          tma_load_3d_hint(sa + C::A_BYTES, &tmB, full, kb * BK, t.n_tile * BN, t.e, tstart[t.e + 1] - tstart[t.e] == 1 ? pol_first : pol_normal);
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok) {
      // let the copies already issued land before the CTA retires its shared memory
      const uint32_t first = issued > (uint32_t)STAGES ? issued - STAGES : 0;
      for (uint32_t j = first; j < issued; ++j) mbar_wait_drain(full0 + 8 * (j % STAGES), (j / STAGES) & 1, DRAIN_LIMIT_NS);
    }
  } else if (warp == 1) {
    // ===================================================================== MMA issuer
    constexpr uint32_t idesc = make_idesc(BM, BN);
    const uint64_t adesc0 = make_smem_desc(smem_u32(smem)), bdesc0 = make_smem_desc(smem_u32(smem) + C::A_BYTES);
    const uint32_t elected = elect_lane();
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(full0 + 8 * stage, phase, abort_flag, p.status, 33)) { ok = false; break; }
        if (!mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1, abort_flag, p.status, 32)) { ok = false; break; }
        tc_fence_after();
        const uint64_t adesc = adesc0 + (uint64_t)(stage * (C::STAGE_BYTES >> 4)), bdesc = bdesc0 + (uint64_t)(stage * (C::STAGE_BYTES >> 4));
        const uint32_t d = tmem_base + (uint32_t)(acc * BN);
#pragma unroll
        for (int k = 0; k < BK / UMMA_K; ++k)       // 32 bytes further inside the swizzle row: +2 in the (addr >> 4) field
          umma_e4m3(elected, d, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc, k != 0 ? 1u : 0u);
        umma_commit_elected(elected, tfull0 + 8 * acc);
        umma_commit_elected(elected, empty0 + 8 * stage);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
    if (!ok) {
      // wait (bounded) until the tensor-core work issued so far has retired, so that tensor memory can be freed
      umma_commit_elected(elected, drain_bar);
      mbar_wait_drain(drain_bar, 0, DRAIN_LIMIT_NS);
    }
  } else {
    // ===================================================================== scaled accumulation and store (warps 2..9)
    const int q = warp & 3;                           // tensor-memory lane quarter this warp may read
    const int half = (warp - 2) >> 2;                 // its half of the columns
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < total_tiles; tile += tile_step) {
      // this thread's scales, and as little else as possible: the accumulators leave hardly any register for the loop
      const float *sa = p.sa + kb0 * p.sa_k, *sb;
      bool any_row;                                   // rows of the warp that are the group's: without one there is nothing to add
      {
        const Tile t = decode_tile(tile, tstart, offs, E, NT);
        const int row = t.row0 + q * 32 + lane;
        if (row < t.row_end) sa += (int64_t)row * p.sa_row;
        any_row = t.row0 + q * 32 < t.row_end;
        // columns behind N have no scale block of their own: the last one stands in, nothing of them is stored
        sb = p.sb + ((int64_t)t.e * p.n_blocks + min((t.n_tile * BN + half * COLS) / 128, p.n_blocks - 1)) * p.k_blocks + kb0;
      }
      f32x2 acc[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) acc[j] = 0ull;
      // the scales of the next block are on their way while this one is added: their product waits for its turn, because taking
      // it at once would hold the warp for the latency of the loads in every block
      float a_next = *sa, b_next = *sb;
      for (int kb = kb0; kb < kb1; ++kb) {
        const float s = a_next * b_next;
        const bool far = __any_sync(0xFFFFFFFFu, no_normal_number(s)) && any_row;
        if (kb + 1 < kb1) {
          sa += p.sa_k;
          ++sb;
          a_next = *sa;
          b_next = *sb;
        }
        if (!mbar_wait_inline(tfull0 + 8 * buf, buf_phase, abort_flag, p.status, 34)) { ok = false; break; }
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + half * COLS);
        if (far) {
          // Read again: keeping both scales would cost every block two registers.  8192 x 4096 x 7168 us: no check 228.4, with it 231.7,
          // every block here (scales of zero come here too) 285.  The product applied to tensor memory in place instead of this
          // second form of the additions: 242 to 264 for ordinary blocks.
          float pre, post;
          split_scale(kb + 1 < kb1 ? *(sa - p.sa_k) : *sa, kb + 1 < kb1 ? *(sb - 1) : *sb, pre, post);
          const f32x2 pre2 = pair_of(pre, pre), post2 = pair_of(post, post);
#pragma unroll
          for (int c = 0; c < COLS / 16; ++c) {
            f32x2 v[8];
            tmem_ld16_pairs(taddr + c * 16, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) fma2(acc[c * 8 + j], mul2(v[j], pre2), post2);
          }
        } else if (any_row) {
          const f32x2 s2 = pair_of(s, s);
#pragma unroll
          for (int c = 0; c < COLS / 16; ++c) {
            f32x2 v[8];
            tmem_ld16_pairs(taddr + c * 16, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) fma2(acc[c * 8 + j], v[j], s2);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty0 + 8 * buf);
        if (++buf == 2) { buf = 0; buf_phase ^= 1; }
      }
      const Tile t = decode_tile(tile, tstart, offs, E, NT);
      if (SPLIT) {
        // every stage has been consumed by the time the last accumulator was ready: the partial tile may take their place
        float* mine = reinterpret_cast<float*>(smem) + (q * 32 + lane) * C::PART_PITCH + half * COLS;
#pragma unroll
        for (int j = 0; j < COLS / 2; j += 2)
          if (t.row0 + q * 32 + lane < t.row_end) *reinterpret_cast<ulonglong2*>(mine + 2 * j) = make_ulonglong2(acc[j], acc[j + 1]);
      } else if (ok) {
        store_rows<COLS>(p, t.row0 + q * 32, t.row_end, lane, t.n_tile * BN + half * COLS, acc,
                         reinterpret_cast<float*>(smem + C::STAGING_OFFSET) + (warp - 2) * 32 * STAGING_PITCH);
      }
    }
    if (p.zero_tail) zero_rows(p, offs[0], offs[E], (int64_t)blockIdx.x * EPI_WARPS + (warp - 2), (int64_t)gridDim.x * EPI_WARPS, lane);
  }

  if (SPLIT) {
    __syncthreads();
    cluster_barrier();
    if (first_tile < total_tiles && threadIdx.x < 256 && !*abort_flag) {
      const Tile t = decode_tile(first_tile, tstart, offs, E, NT);
      const int live = min(BM, t.row_end - t.row0);
      for (int i = rank * 256 + threadIdx.x; i < live * (BN / 4); i += S * 256) {
        const int r = i / (BN / 4), c = (i - r * (BN / 4)) * 4;
        const uint32_t at = smem_u32(smem) + (uint32_t)(r * C::PART_PITCH + c) * 4;
        float4 v[MAX_SPLIT];
#pragma unroll
        for (int s = 0; s < MAX_SPLIT; ++s)
          if (s < S) v[s] = ld_cluster(map_to_cta(at, s));
        float4 sum = v[0];
#pragma unroll
        for (int s = 1; s < MAX_SPLIT; ++s)
          if (s < S) { sum.x += v[s].x; sum.y += v[s].y; sum.z += v[s].z; sum.w += v[s].w; }
        store_four(p, t.row0 + r, t.n_tile * BN + c, sum);
      }
    }
    cluster_barrier();        // nobody leaves while its partial tile is still read
  }

  // ---- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------ host side
// 8-bit tensor [d2][d1][d0] (d0 contiguous, rows ld1 bytes apart), box [1][box1][128], 128-byte swizzle, zeros out of bounds
static int make_tmap8(CUtensorMap* m, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t ld1, uint32_t box1) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return fail(MOE_ERR_DEVICE, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {ld1, ld1 * d1};
  cuuint32_t box[3] = {(cuuint32_t)BK, box1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, d2 > 0 ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(MOE_ERR_ARG, "cuTensorMapEncodeTiled failed with %d (dims %llu,%llu,%llu row %llu box1 %u)", (int)r, (unsigned long long)d0,
                (unsigned long long)d1, (unsigned long long)d2, (unsigned long long)ld1, box1);
  return MOE_OK;
}

// split: CTAs per cluster, or 1
template <int BN, bool SPLIT, int AR>
static int launch(const void* A, int64_t lda, const void* B, Params p, int64_t tiles, int split, int sms, cudaStream_t st) {
  using C = Cfg<BN, AR>;
  auto kernel = fp8_gemm_kernel<BN, SPLIT, AR>;
  static std::atomic<bool> attr_set[64];
  int rc = allow_dynamic_smem(kernel, C::SMEM_BYTES, attr_set);
  if (rc) return rc;
  p.n_tiles = (p.N + BN - 1) / BN;
  CUtensorMap tA, tAFew, tB;
  rc = make_tmap8(&tA, A, (uint64_t)p.K, (uint64_t)p.rows, 0, (uint64_t)lda, (uint32_t)p.a_box_rows);
  if (rc) return rc;
  rc = make_tmap8(&tAFew, A, (uint64_t)p.K, (uint64_t)p.rows, 0, (uint64_t)lda, (uint32_t)FEW_ROWS);
  if (rc) return rc;
  rc = make_tmap8(&tB, B, (uint64_t)p.K, (uint64_t)p.N, (uint64_t)p.E, (uint64_t)p.K, (uint32_t)BN);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(SPLIT ? tiles * split : (tiles < sms ? tiles : sms)), 1, 1);
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 1 : 0;
  MOE_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, tA, tAFew, tB, p));
  return MOE_OK;
}

}  // namespace gemm8
}  // namespace moe

// ====================================================================================
extern "C" int moe_fp8_gemm(const void* A, int64_t lda, const float* a_scale, int64_t as_row, int64_t as_k, const void* B,
                            const float* b_scale, const int32_t* offsets, int64_t rows, int K, int N, int E, void* Y, int64_t ldy,
                            int out_dtype, int zero_tail, int32_t* status, void* stream) {
  using namespace moe;
  using namespace moe::gemm8;
  if (out_dtype < 0 || out_dtype > MOE_DTYPE_F32) return fail(MOE_ERR_ARG, "fp8_gemm: unknown output type %d", out_dtype);
  if (rows < 0 || K < 16 || K % 16 || N < 1 || E < 1)
    return fail(MOE_ERR_ARG, "fp8_gemm: bad shape rows=%lld K=%d N=%d E=%d (K a multiple of 16)", (long long)rows, K, N, E);
  if (K > 0x7FFF0000 || N > 0x7FFF0000) return fail(MOE_ERR_UNSUPPORTED, "fp8_gemm: K=%d or N=%d too wide", K, N);
  if (E > MAX_E) return fail(MOE_ERR_UNSUPPORTED, "fp8_gemm: E=%d exceeds %d", E, MAX_E);
  if (!offsets && E != 1) return fail(MOE_ERR_ARG, "fp8_gemm: several groups need an offsets table");
  if (rows == 0) return MOE_OK;
  if (rows > 0x7FFFFF00ll) return fail(MOE_ERR_UNSUPPORTED, "fp8_gemm: too many rows");
  if (!A || !a_scale || !B || !b_scale || !Y) return fail(MOE_ERR_ARG, "fp8_gemm: null pointer");
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) return fail(MOE_ERR_ARG, "fp8_gemm: A and B must be 16-byte aligned");
  if (lda < K || lda % 16) return fail(MOE_ERR_ARG, "fp8_gemm: lda=%lld must be at least K and a multiple of 16", (long long)lda);
  if (as_row < 0 || as_k < 0) return fail(MOE_ERR_ARG, "fp8_gemm: negative stride of the row scales");
  if (ldy < N) return fail(MOE_ERR_ARG, "fp8_gemm: ldy=%lld is less than N", (long long)ldy);
  DeviceInfo dev;
  int rc = current_device_info(&dev);
  if (rc) return rc;
  Params p;
  p.sa = a_scale; p.sa_row = as_row; p.sa_k = as_k; p.sb = b_scale; p.offsets = offsets;
  p.Y = Y; p.ldy = ldy; p.rows = (int)rows; p.K = K; p.N = N; p.E = E;
  p.n_tiles = 0; p.k_blocks = (K + BK - 1) / BK; p.n_blocks = (N + 127) / 128;
  p.out = out_dtype; p.zero_tail = zero_tail != 0 && offsets != nullptr; p.status = status;
  const int64_t el = out_dtype == MOE_DTYPE_F32 ? 4 : 2;
  p.vec_store = !(reinterpret_cast<uintptr_t>(Y) & 15) && (ldy * el) % 16 == 0 && (N * el) % 16 == 0;
  if (p.vec_store && !(reinterpret_cast<uintptr_t>(Y) & 31) && (ldy * el) % 32 == 0 && (N * el) % 32 == 0) p.vec_store = 2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // Tiles of 256 or of 128 columns: a round of the wider takes about 3 / 2 the time of one of the narrower (us, wide / narrow:
  // 512 x 4096 x 4096, one round each, 21.4 / 16.0; 2500 x 2048 x 2048, two and three, 23.5 / 23.4; 1024 x 4096 x 4096, one and two, 21.8 /
  // 27.1), and the launch as many rounds of tiles as the SMs need.  Where even the narrow tiles leave SMs idle, clusters of 2, 4
  // or 8 CTAs share the k-blocks of a tile (clusters of 4 and 8 do not fill the GPU: counted as 128 SMs), two k-blocks each at
  // least.  A token through 4096 x 7168: 35 us on 16 wide tiles, 11.8 on 32 clusters of 4.
  const int64_t m_tiles = offsets ? rows / BM + (rows < E ? rows : E) : ceil_div64(rows, BM);
  const int64_t tiles256 = m_tiles * ceil_div64(N, 256), tiles128 = m_tiles * ceil_div64(N, 128);
  if (tiles128 > 0x7FFFFFFFll) return fail(MOE_ERR_UNSUPPORTED, "fp8_gemm: too many tiles");
  p.a_box_rows = rows < BM ? (int)(rows + 7) / 8 * 8 : BM;
  if (ceil_div64(tiles256, dev.sm_count) * 3 <= ceil_div64(tiles128, dev.sm_count) * 2)
    return launch<256, false, BM>(A, lda, B, p, tiles256, 1, dev.sm_count, st);
  int split = 1;
  while (split < MAX_SPLIT && p.k_blocks >= 4 * split && tiles128 * split * 2 <= (split == 1 ? dev.sm_count : dev.sm_count * 7 / 8)) split *= 2;
  if (rows <= FEW_ROWS)      // nearly all of the ring holds weights then: a token through 4096 x 7168, weights in L2, 11.8 -> 10.1 us
    return split > 1 ? launch<128, true, FEW_ROWS>(A, lda, B, p, tiles128, split, dev.sm_count, st)
                     : launch<128, false, FEW_ROWS>(A, lda, B, p, tiles128, 1, dev.sm_count, st);
  return split > 1 ? launch<128, true, BM>(A, lda, B, p, tiles128, split, dev.sm_count, st)
                   : launch<128, false, BM>(A, lda, B, p, tiles128, 1, dev.sm_count, st);
}
