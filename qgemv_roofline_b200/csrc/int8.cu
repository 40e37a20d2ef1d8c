// int8 matrix products with one scale per token and one per channel:
//   y[n][m] = (sum_k xq[n][k] wq[m][k]) * xs[n] * ws[m] (+ bias[m])
// and the rounding of activations to int8 with one scale per row:
//   xs = max |x| / 127,  xq = rint(x / xs).
//
// The sum is exact: tcgen05.mma kind::i8 accumulates in int32, which holds
// K * 128 * 128 for K below 2^17 (larger K is refused).  It becomes fp32 once,
// is multiplied by the token's scale, then by the channel's with the bias added
// in the same operation, and the result is rounded to y's type: three roundings
// to fp32, then y's.
//
// Weights take the MMA's M side (128 channels per CTA), tokens its N side.
// Both operands are K-major int8 rows, copied by TMA as boxes of 128 bytes
// with 128-byte swizzle, the layout the tensor core reads; rows and columns
// past the end read as zeros.  TMEM lane = channel, column = token: a warp
// stores 32 consecutive channels of a token at a time.  Two kernels:
//
//  * k_int8_mm (up to 128 tokens, more with few tiles): one tile of 128 channels
//    x 16 to 128 tokens per CTA or, where the tiles leave room, per cluster, whose
//    CTAs split K and add their int32 parts through distributed shared memory
//    (exact in any order).  With one token the weights' stream is what counts.
//  * k_int8_pair (more): persistent CTA pairs (tcgen05 cta_group::2) on tiles of
//    256 channels x up to 256 tokens; each CTA copies its half of both operands, so
//    that an SM reads 64 instead of 96 bytes of shared memory per cycle; two
//    accumulators in TMEM, so that one tile is stored while the next is summed.
#include <algorithm>
#include <cstring>

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "qgemv_common.cuh"
#include "qgemv_internal.h"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace qg {

__device__ int g_i8_error = 0;
__device__ long long g_i8_spin_limit = kDefaultSpinLimit;

namespace {

constexpr int I8_M = 128;        // channels per tile
constexpr int I8_KB = 128;       // bytes (= columns) of a K step
constexpr int I8_ABYTES = I8_M * I8_KB;
constexpr int I8_THREADS = 192;  // producer, MMA, 4 epilogue warps

__device__ __forceinline__ long long i8_spin_limit() {
  return *(volatile long long*)&g_i8_spin_limit;
}
// Bounded wait; gives up at once when another thread raised the abort flag.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64(), lim = i8_spin_limit();
  while (!mbar_try(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > lim) {
      atomicExch(&g_i8_error, (int)ERR_TIMEOUT);
      __threadfence();
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// The same by a whole warp, which goes on or gives up as one: a lane may see
// the barrier, another the abort flag, and what follows (elections, TMEM loads,
// shuffles, barriers of the CTA) wants every lane.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// Wait for copies and MMAs in flight before the CTA exits (they complete on
// their own): ignores the abort flag, bounded by at least the default limit.
__device__ __forceinline__ void mbar_wait_drain(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64(), lim = max(i8_spin_limit(), kDefaultSpinLimit);
  while (!mbar_try(bar, parity) && clock64() - t0 < lim) {
  }
}

// ------------------------------------------------------------- row scales
template <typename T> __device__ __forceinline__ float as_f32(T v) { return (float)v; }
template <> __device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// q = rint(x / s), the quotient rounded to fp32 first, in the low byte.  x * (1 / s)
// is within 127 * 2^-22 of the quotient, so only where it comes that near to a
// tie (or where 1 / s is not accurate) is the division itself needed.  Adding
// 1.5 * 2^23 rounds to an integer, half to even, which is then the low bits of
// the sum: no conversion instruction (16 a clock per SM, and there were two).
__device__ __forceinline__ uint32_t quant_near(float v, float inv, bool& tie) {
  const float r = v * inv, t = r + 12582912.0f;
  tie |= fabsf(fabsf(r - (t - 12582912.0f)) - 0.5f) < 6.2e-5f;
  return __float_as_uint(t);
}
__device__ __noinline__ uint32_t quant_exact(float v, float s) {
  return (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.0f), 127.0f);
}

constexpr int RQ_THREADS = 256;
constexpr int RQ_HELD = 2;  // vectors of 8 values that a thread keeps

// One CTA per row.  4096 rows of 4096 in bf16: 16.4 us (50 MB, 7.7 at the copy
// rate), 2.8 of 4 instructions per cycle with half the warps: issue and, at the
// barrier between reading and writing, the loads' latency.  A single row is a
// launch and two round trips (4.8 us alone).  A row with a NaN or an infinity gets the scale NaN and
// zeros; an all-zero row (or one whose scale underflows to 0) the scale 0 and
// zeros.  VEC: rows start on 16-byte boundaries, q's on 8-byte ones, and K is a
// multiple of 8: a row of up to 4096 values is read once and kept.
template <typename T, bool VEC>
__global__ void __launch_bounds__(RQ_THREADS) k_quant_rows(const T* __restrict__ x, int64_t ldx, int K,
                                                           int8_t* __restrict__ q, int64_t ldq,
                                                           float* __restrict__ s) {
  __shared__ uint32_t red[RQ_THREADS / 32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  int8_t* qr = q + row * ldq;
  // 8 values as they are read (kept so, for registers: the kernel is many short
  // CTAs, and 64 registers a thread halved how many an SM holds)
  struct Raw {
    uint4 u[sizeof(T) / 2];
  };
  auto load8 = [&](Raw& r, int i) {  // values 8 i ...
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) r.u[j] = reinterpret_cast<const uint4*>(xr)[i * (int)(sizeof(T) / 2) + j];
  };
  auto value = [](const Raw& r, int j) { return as_f32(reinterpret_cast<const T*>(&r)[j]); };
  auto bits = [](float v) { return __float_as_uint(v) & 0x7FFFFFFFu; };
  uint32_t m = 0u;
  Raw held[RQ_HELD];
  const int nv = K / 8;
  if (VEC) {
#pragma unroll
    for (int h = 0; h < RQ_HELD; ++h)
      if (threadIdx.x + h * RQ_THREADS < nv) load8(held[h], threadIdx.x + h * RQ_THREADS);
#pragma unroll
    for (int h = 0; h < RQ_HELD; ++h)
      if (threadIdx.x + h * RQ_THREADS < nv)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, bits(value(held[h], j)));
    for (int i = threadIdx.x + RQ_HELD * RQ_THREADS; i < nv; i += RQ_THREADS) {
      Raw v;
      load8(v, i);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, bits(value(v, j)));
    }
  } else {
    for (int k = threadIdx.x; k < K; k += RQ_THREADS) m = max(m, bits(as_f32(xr[k])));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RQ_THREADS / 32; ++i) m = max(m, red[i]);
  const bool bad = m >= 0x7F800000u;
  const float sc = bad ? __int_as_float(0x7FC00000) : __fdiv_rn(__uint_as_float(m), 127.0f);
  const bool some = sc > 0.0f, exact = sc < 7.9e-31f;  // 2^-100: 1 / s stays a normal number above
  const float inv = some ? __fdiv_rn(1.0f, sc) : 0.0f;
  if (threadIdx.x == 0) s[row] = sc;
  if (VEC) {
    auto put8 = [&](const Raw& v, int i) {
      uint32_t w[2] = {0u, 0u};
      if (some) {
        uint32_t b[8];
        bool tie = exact;
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = quant_near(value(v, j), inv, tie);
        if (tie)
          for (int j = 0; j < 8; ++j) b[j] = quant_exact(value(v, j), sc);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[j] = __byte_perm(__byte_perm(b[4 * j], b[4 * j + 1], 0x0040), __byte_perm(b[4 * j + 2], b[4 * j + 3], 0x0040),
                             0x5410);
      }
      reinterpret_cast<uint2*>(qr)[i] = make_uint2(w[0], w[1]);
    };
#pragma unroll
    for (int h = 0; h < RQ_HELD; ++h) {
      const int i = threadIdx.x + h * RQ_THREADS;
      if (i < nv) put8(held[h], i);
    }
    for (int i = threadIdx.x + RQ_HELD * RQ_THREADS; i < nv; i += RQ_THREADS) {
      Raw v;
      load8(v, i);
      put8(v, i);
    }
  } else {
    for (int k = threadIdx.x; k < K; k += RQ_THREADS)
      qr[k] = some ? (int8_t)quant_exact(as_f32(xr[k]), sc) : (int8_t)0;
  }
}

// ---------------------------------------------------------------- product
struct I8Args {
  alignas(64) CUtensorMap wmap;  // [M][K] int8, boxes of 128 bytes x 128 rows
  alignas(64) CUtensorMap xmap;  // [N][K] int8, boxes of 128 bytes x BN (pairs: 128) rows
  const float* xs;
  const float* ws;
  const float* bias;
  void* y;
  int64_t ldy;
  int M, N, nk;    // nk: K steps
  // The weights may be read before the dependency wait: the launch before this
  // one is the row kernel of the same call, every CTA of which had waited for
  // what came before it when this launch was allowed; the copies read L2, where
  // those writes are by then.
  int early_w;
};

constexpr int I8_CL = 8;  // CTAs of a cluster at most

// BN tokens per tile; S ring stages.  kind::i8: s32 accumulators (bits 4-5 =
// 2), A and B signed (bits 7-9, 10-12 = 1), both K-major, N >> 3 at bit 17,
// M >> 4 at bit 24.
template <int BN>
struct I8Cfg {
  static constexpr int STAGE = I8_ABYTES + BN * I8_KB;
  static constexpr int S = BN == 128 ? 3 : 4;
  static constexpr int COLS = BN < 32 ? 32 : BN;  // TMEM columns
  static constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) |
                                    ((uint32_t)(I8_M >> 4) << 24);
  static constexpr size_t SMEM = (size_t)S * STAGE + 1024;
};

__device__ __forceinline__ void put_y(float* y, float v) { *y = v; }
__device__ __forceinline__ void put_y(__nv_bfloat16* y, float v) { *y = __float2bfloat16(v); }
__device__ __forceinline__ void put_y(__half* y, float v) { *y = __float2half(v); }
// two channels of one token
__device__ __forceinline__ void put_y2(__nv_bfloat16* y, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(y) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void put_y2(__half* y, float a, float b) {
  *reinterpret_cast<__half2*>(y) = __floats2half2_rn(a, b);
}

// Four channels of one token, `room` of them exist; one store where `vec`.
__device__ __forceinline__ void put_y4(float* y, const float (&f)[4], int room, bool vec) {
  if (vec && room >= 4) {
    *reinterpret_cast<float4*>(y) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < room) y[i] = f[i];
  }
}
template <typename Y>
__device__ __forceinline__ void put_y4(Y* y, const float (&f)[4], int room, bool vec) {
  if (vec && room >= 4) {
    __align__(8) Y h[4];
    put_y2(h, f[0], f[1]);
    put_y2(h + 2, f[2], f[3]);
    *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(h);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < room) put_y(y + i, f[i]);
  }
}

// NC accumulator columns (tokens) from `ta` on, this lane's channel: scaled and
// stored; `nn` of them exist.  xs: their scales in shared memory.  y: token 0's
// element of the warp's first channel; `room`: channels from there on.  With a
// 16-bit type and even addresses a pair of lanes trades values, so that one
// store writes two channels of one token in the even lane and of the next in the
// odd one: half the stores of one value each, and no 2-byte ones.
template <typename Y, int NC>
__device__ __forceinline__ void store_cols(uint32_t ta, int nn, const float* xs, float ws, float b, Y* y,
                                           int64_t ldy, int room, int lane) {
  constexpr int STEP = NC < 32 ? 16 : 32;
  const bool pairs = sizeof(Y) == 2 && room >= 32 && (reinterpret_cast<uintptr_t>(y) & 3) == 0 && (ldy & 1) == 0;
  const bool odd = lane & 1;
#pragma unroll 1
  for (int c = 0; c < NC && c < nn; c += STEP) {
    uint32_t v[STEP];
    if constexpr (STEP == 16) tmem_ld<16>(ta + c, v);
    else tmem_ld32(ta + c, v);
    tmem_ld_wait();
    Y* p = y + (int64_t)c * ldy;
    if (sizeof(Y) == 2 && pairs && c + STEP <= nn) {
      if constexpr (sizeof(Y) == 2) {
        p += (lane & ~1) + (odd ? ldy : 0);
#pragma unroll
        for (int j = 0; j < STEP; j += 4, p += 4 * ldy) {
          const float4 s = *reinterpret_cast<const float4*>(xs + c + j);
          const float f0 = fmaf((float)(int)v[j] * s.x, ws, b), f1 = fmaf((float)(int)v[j + 1] * s.y, ws, b);
          const float f2 = fmaf((float)(int)v[j + 2] * s.z, ws, b), f3 = fmaf((float)(int)v[j + 3] * s.w, ws, b);
          const float g = __shfl_xor_sync(0xffffffffu, odd ? f0 : f1, 1);
          const float h = __shfl_xor_sync(0xffffffffu, odd ? f2 : f3, 1);
          put_y2(p, odd ? g : f0, odd ? f1 : g);
          put_y2(p + 2 * ldy, odd ? h : f2, odd ? f3 : h);
        }
      }
    } else {
      p += lane;
#pragma unroll
      for (int j = 0; j < STEP; ++j, p += ldy)
        if (c + j < nn && lane < room) put_y(p, fmaf((float)(int)v[j] * xs[c + j], ws, b));
    }
  }
}

// Grid (channel tiles x cluster size, token tiles).  The CTAs of a cluster
// split the K steps of one tile; their int32 parts are added through
// distributed shared memory (exact, so in any order).
template <int BN, typename Y>
__global__ void __launch_bounds__(I8_THREADS) k_int8_mm(const __grid_constant__ I8Args p) {
  using C = I8Cfg<BN>;
  constexpr int S = C::S;
  extern __shared__ uint8_t i8_smem_raw[];
  __shared__ __align__(8) unsigned long long full[S], empty[S], done;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ __align__(16) float xs_s[BN];
  cg::cluster_group cl = cg::this_cluster();
  Y* y = static_cast<Y*>(p.y);
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(i8_smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t ring_s = saddr(ring);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = (int)(blockIdx.x / cs) * I8_M, n0 = (int)blockIdx.y * BN;
  const int k0 = (int)((int64_t)p.nk * rank / cs), steps = (int)((int64_t)p.nk * (rank + 1) / cs) - k0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(saddr(&full[s]), 1);
      mbar_init(saddr(&empty[s]), 1);
    }
    mbar_init(saddr(&done), 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     saddr(&tmem_base)),
                 "r"(C::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  // the producer and the MMA warp run their loops as a whole, one elected lane
  // issues: addresses and descriptors are then in uniform registers
  if (warp == 0) {
    {
      const int pre = min(S, steps);
      auto load_w = [&](int i) {
        if (elect_one()) {
          mbar_expect_tx(saddr(&full[i % S]), C::STAGE);
          tensor_g2s(ring_s + (i % S) * C::STAGE, &p.wmap, (k0 + i) * I8_KB, m0, saddr(&full[i % S]));
        }
      };
      auto load_x = [&](int i) {
        if (elect_one())
          tensor_g2s(ring_s + (i % S) * C::STAGE + I8_ABYTES, &p.xmap, (k0 + i) * I8_KB, n0,
                     saddr(&full[i % S]));
      };
      if (p.early_w)
        for (int i = 0; i < pre; ++i) load_w(i);
      pdl_wait();
      if (!p.early_w)
        for (int i = 0; i < pre; ++i) load_w(i);
      for (int i = 0; i < pre; ++i) load_x(i);
      int issued = pre;
      for (int i = pre; i < steps; ++i) {
        if (!warp_wait(saddr(&empty[i % S]), (uint32_t)((i / S - 1) & 1), &abort_flag)) break;
        load_w(i);
        load_x(i);
        issued = i + 1;
      }
      // no copy outlives the CTA, whatever the other warps gave up on
      for (int i = max(0, issued - S); i < issued; ++i)
        mbar_wait_drain(saddr(&full[i % S]), (uint32_t)((i / S) & 1));
    }
  } else if (warp == 1) {
    pdl_wait();  // so that the bounded waits below do not count the previous kernel's time
    bool ok = true;
    for (int i = 0; i < steps && ok; ++i) {
      const int s = i % S;
      ok = warp_wait(saddr(&full[s]), (uint32_t)((i / S) & 1), &abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t da = sw128_desc(ring_s + s * C::STAGE), db = sw128_desc(ring_s + s * C::STAGE + I8_ABYTES);
#pragma unroll
        for (int k = 0; k < I8_KB / 32; ++k)
          tc_mma_i8<1>(tmem, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), C::IDESC, i > 0 || k > 0);
        tc_commit(saddr(&empty[s]));
      }
      __syncwarp();
    }
    if (elect_one()) tc_commit(saddr(&done));
    __syncwarp();
    mbar_wait_drain(saddr(&done), 0u);  // no MMA outlives its operands or the accumulators
  } else {
    pdl_wait();  // xs
    if (warp == 2) pdl_trigger();
    const int nn = min(BN, p.N - n0);
    const int quarter = warp & 3, row = quarter * 32 + lane, m = m0 + row;
    for (int c = threadIdx.x - 64; c < nn; c += 128) xs_s[c] = p.xs[n0 + c];
    const float ws = m < p.M ? p.ws[m] : 0.0f, b = m < p.M && p.bias ? p.bias[m] : 0.0f;
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the four epilogue warps
    warp_wait(saddr(&done), 0u, &abort_flag);  // given up or not: the rest is in bounds
    tc_fence_after();
    const uint32_t ta = tmem + ((uint32_t)(quarter * 32) << 16);
    if (cs > 1) {
      int* part = reinterpret_cast<int*>(ring);  // [BN][128], once the ring is idle (done)
      for (int c = 0; c < nn; c += 16) {
        uint32_t v[16];
        tmem_ld<16>(ta + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * I8_M + row] = (int)v[j];
      }
    } else {
      store_cols<Y, BN>(ta, nn, xs_s, ws, b, y + (int64_t)n0 * p.ldy + m - lane, p.ldy, p.M - m + lane, lane);
    }
  }
  __syncwarp();
  if (cs > 1) {
    // A warp joins one token's 128 channels, four a lane, all parts in flight at
    // once: a part is another SM's shared memory, so each read is a long
    // latency and few bytes (128 tokens, 4096 -> 11008: one value a thread at a
    // time 30.6 us, now 16.5 with the same two CTAs a tile)
    const int nn = min(BN, p.N - n0), m = m0 + 4 * lane, room = p.M - m;
    float ws[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ws[i] = i < room ? p.ws[m + i] : 0.0f;
      b[i] = i < room && p.bias ? p.bias[m + i] : 0.0f;
    }
    const bool vec = (reinterpret_cast<uintptr_t>(p.y) & (4 * sizeof(Y) - 1)) == 0 && (p.ldy & 3) == 0;
    const int4* part[I8_CL];
#pragma unroll
    for (int r = 0; r < I8_CL; ++r)
      part[r] = reinterpret_cast<const int4*>(cl.map_shared_rank(reinterpret_cast<int*>(ring), min(r, cs - 1)));
    cl.sync();
    for (int c = rank + cs * warp; c < nn; c += cs * (I8_THREADS / 32)) {
      int4 v[I8_CL];
#pragma unroll
      for (int r = 0; r < I8_CL; ++r) v[r] = r < cs ? part[r][c * (I8_M / 4) + lane] : make_int4(0, 0, 0, 0);
      int s[4] = {};
#pragma unroll
      for (int r = 0; r < I8_CL; ++r) s[0] += v[r].x, s[1] += v[r].y, s[2] += v[r].z, s[3] += v[r].w;
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = fmaf((float)s[i] * xs_s[c], ws[i], b[i]);
      put_y4(y + (int64_t)(n0 + c) * p.ldy + m, f, room, vec);
    }
    cl.sync();  // no CTA leaves while another reads its part
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS)
                 : "memory");
  }
}

// ----------------------------------------------------------- CTA pairs
constexpr int PR_N = 256;                             // tokens per tile, at most
constexpr int PR_STAGE = I8_ABYTES + (PR_N / 2) * I8_KB;  // a CTA's half: up to 32 KB
constexpr int PR_S = 6;
constexpr int PR_EW = 8;                              // epilogue warps
constexpr int PR_THREADS = 32 * (2 + PR_EW);
constexpr size_t PR_SMEM = (size_t)PR_S * PR_STAGE + 1024;

// Tiles t = cluster, cluster + clusters, ... of (channel tile t / token tiles,
// token tile t % token tiles): tiles under way at the same time share channel
// tiles, and all token tiles stay in L2.  CTA 0 of the pair issues the MMAs; the
// copies of both CTAs complete on CTA 0's `full` barriers, and its commits
// arrive on both CTAs' `empty` and `tfull` barriers.  `width` tokens per tile
// (a multiple of 32): what fills the pairs best.
template <typename Y>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PR_THREADS, 1)
    k_int8_pair(const __grid_constant__ I8Args p, int width, int ntn, int tiles) {
  extern __shared__ uint8_t pr_smem_raw[];
  __shared__ __align__(8) unsigned long long full[PR_S], empty[PR_S], tfull[2], tempty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ __align__(16) float xs_s[PR_EW][PR_N / 2];
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t rank = cl.block_rank();
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(pr_smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t ring_s = saddr(ring);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2, hw = width / 2;
  const int mine = pair < tiles ? (tiles - pair + pairs - 1) / pairs : 0;  // tiles of this pair
  if (threadIdx.x == 0) {
    for (int s = 0; s < PR_S; ++s) {
      mbar_init(saddr(&full[s]), 1);
      mbar_init(saddr(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(saddr(&tfull[b]), 1);
      mbar_init(saddr(&tempty[b]), 2 * PR_EW);  // both CTAs' epilogue warps
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     saddr(&tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cl.sync();  // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    {
      // a step at a time: K step k of tile t into stage s (counted, not divided:
      // one thread does all this, in the time of four MMAs)
      struct At {
        int s, k, t;
      };
      const uint32_t fbar = cluster_addr(saddr(&full[0]), 0);
      auto next = [&](At& at) {
        if (++at.s == PR_S) at.s = 0;
        if (++at.k == p.nk) {
          at.k = 0;
          at.t += pairs;
        }
      };
      auto load_w = [&](const At& at, int m0) {
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(saddr(&full[at.s]), 2 * (uint32_t)(I8_ABYTES + hw * I8_KB));
          tensor_g2s_pair(ring_s + at.s * PR_STAGE, &p.wmap, at.k * I8_KB, m0, fbar + 8 * at.s);
        }
      };
      auto load_x = [&](const At& at, int n0) {
        if (elect_one())
          tensor_g2s_pair(ring_s + at.s * PR_STAGE + I8_ABYTES, &p.xmap, at.k * I8_KB, n0, fbar + 8 * at.s);
      };
      auto m_of = [&](int t) { return (t / ntn) * 2 * I8_M + (int)rank * I8_M; };
      auto n_of = [&](int t) { return (t % ntn) * width + (int)rank * hw; };
      const int64_t total = (int64_t)mine * p.nk;
      const int pre = (int)min((int64_t)PR_S, total);
      At at{0, 0, pair};
      if (p.early_w)
        for (int i = 0; i < pre; ++i, next(at)) load_w(at, m_of(at.t));
      pdl_wait();
      at = At{0, 0, pair};
      for (int i = 0; i < pre; ++i, next(at)) {
        if (!p.early_w) load_w(at, m_of(at.t));
        load_x(at, n_of(at.t));
      }
      int64_t issued = pre;
      uint32_t phase = 0u;
      int m0 = m_of(at.t), n0 = n_of(at.t);
      while (issued < total) {
        if (!warp_wait(saddr(&empty[at.s]), phase, &abort_flag)) break;
        if (at.k == 0) {
          m0 = m_of(at.t);
          n0 = n_of(at.t);
        }
        load_w(at, m0);
        load_x(at, n0);
        next(at);
        if (at.s == 0) phase ^= 1u;
        ++issued;
      }
      // no copy outlives the pair (CTA 1's complete on CTA 0's barriers; the
      // cluster barrier below holds CTA 1 until CTA 0 has seen them)
      if (rank == 0)
        for (int64_t i = max((int64_t)0, issued - PR_S); i < issued; ++i)
          mbar_wait_drain(saddr(&full[i % PR_S]), (uint32_t)((i / PR_S) & 1));
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    // the whole warp runs the loop, one elected lane issues: what an MMA takes is
    // then in uniform registers (a lane's own branch cost more cycles per MMA
    // than narrow tiles' MMAs take)
    if (rank == 0) {
      pdl_wait();  // so that the bounded waits below do not count the previous kernel's time
      const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(width >> 3) << 17) |
                             ((uint32_t)(2 * I8_M >> 4) << 24);
      const uint64_t da0 = sw128_desc(ring_s), db0 = sw128_desc(ring_s + I8_ABYTES);
      bool ok = true;
      int s = 0, t = 0;
      uint32_t phase = 0u;
      for (; t < mine && ok; ++t) {
        const int b = t & 1;
        if (t >= 2) ok = warp_wait(saddr(&tempty[b]), (uint32_t)((t / 2 - 1) & 1), &abort_flag);
        tc_fence_after();
        for (int k = 0; k < p.nk && ok; ++k) {
          ok = warp_wait(saddr(&full[s]), phase, &abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint64_t da = da0 + (uint64_t)(s * (PR_STAGE / 16)), db = db0 + (uint64_t)(s * (PR_STAGE / 16));
#pragma unroll
            for (int kk = 0; kk < I8_KB / 32; ++kk)
              tc_mma_i8<2>(tmem + b * PR_N, da + (uint64_t)(kk * 2), db + (uint64_t)(kk * 2), idesc,
                           k > 0 || kk > 0);
            tc_commit_pair(saddr(&empty[s]));
          }
          __syncwarp();
          if (++s == PR_S) {
            s = 0;
            phase ^= 1u;
          }
        }
        if (ok && elect_one()) tc_commit_pair(saddr(&tfull[b]));
        __syncwarp();
      }
      // no MMA outlives the pair's operands or accumulators: the last commit
      if (ok && mine > 0) {
        mbar_wait_drain(saddr(&tfull[(mine - 1) & 1]), (uint32_t)(((mine - 1) / 2) & 1));
      } else if (!ok) {
        if (elect_one()) tc_commit_pair(saddr(&tfull[t & 1]));
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {  // a launch that gave up: what was issued ends within microseconds
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    pdl_wait();
    if (warp == 2) pdl_trigger();
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    float* xs = xs_s[warp - 2];
    for (int t = 0; t < mine; ++t) {
      const int tile = pair + t * pairs, b = t & 1;
      const int m = (tile / ntn) * 2 * I8_M + (int)rank * I8_M + quarter * 32 + lane;
      const int n0 = (tile % ntn) * width + half * hw, nn = min(hw, p.N - n0);
      __syncwarp();
      for (int c = lane; c < nn; c += 32) xs[c] = p.xs[n0 + c];
      const float ws = m < p.M ? p.ws[m] : 0.0f, bv = m < p.M && p.bias ? p.bias[m] : 0.0f;
      __syncwarp();
      if (!warp_wait(saddr(&tfull[b]), (uint32_t)((t / 2) & 1), &abort_flag)) break;
      tc_fence_after();
      store_cols<Y, PR_N / 2>(tmem + ((uint32_t)(quarter * 32) << 16) + b * PR_N + half * hw, nn, xs, ws, bv,
                              static_cast<Y*>(p.y) + (int64_t)n0 * p.ldy + m - lane, p.ldy, p.M - m + lane, lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(saddr(&tempty[b]), 0));
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cl.sync();  // neither CTA leaves while the pair's copies, MMAs or arrivals reach it
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

template <typename... A>
int launch(const char* what, void (*f)(A...), dim3 grid, int threads, size_t smem, int cluster,
           cudaStream_t st, A... args) {
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, f, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  }
  return OK;
}

// With few tiles a cluster splits the K steps, as many CTAs as are resident at
// once, each with enough steps that its part is worth the join: 2 at 16 columns,
// up to 8 at 64 and more (4096 columns deep, clusters of 1/2/3/4/8: 64 tokens ->
// 11008 13.8/15.0/12.3/17.9/24.3 us, of which 4 and 8 are not resident; 128
// tokens -> 4096 14.7/12.7/10.4/9.7/11.9)
template <int BN, typename Y>
int split_of(int64_t tiles, int nk, const DeviceInfo& dev, int* cs) {
  using C = I8Cfg<BN>;
  const int least = std::min(8, BN / 8);
  // by shared memory (2 KB for what is not dynamic): the occupancy query answers
  // 1 for a kernel that allocates TMEM, though 3 ran at once at 16 columns
  const int per_sm = std::max(1, (int)(dev.smem_optin / (C::SMEM + 2048)));
  const int64_t room = (int64_t)per_sm * dev.sms / tiles;
  *cs = 1;
  for (int t = (int)std::min<int64_t>(std::min<int64_t>(I8_CL, room), nk / least); t > 1; --t) {
    int most = 0;  // with one CTA per SM
    if (int rc = active_clusters((const void*)k_int8_mm<BN, Y>, dev, I8_THREADS, dev.smem_optin - 4096, t, &most))
      return rc;
    if (tiles <= (int64_t)most * per_sm) {
      *cs = t;
      break;
    }
  }
  return OK;
}

template <int BN, typename Y>
int launch_mm(const Int8Call& c, I8Args& a, const DeviceInfo& dev, cudaStream_t st) {
  using C = I8Cfg<BN>;
  if (int rc = allow_max_smem((const void*)k_int8_mm<BN, Y>, dev)) return rc;
  const int tiles = (int)((c.M + I8_M - 1) / I8_M);
  const int64_t step = (int64_t)BN * 65535;  // token tiles of one launch
  for (int64_t n0 = 0; n0 < c.N; n0 += step) {
    const int64_t n = std::min(step, c.N - n0);
    const int64_t nt = (n + BN - 1) / BN;
    if (int rc = encode_tensor_2d(&a.wmap, false, c.wq, c.K, c.M, c.ldw, I8_KB, I8_M, true)) return rc;
    if (int rc = encode_tensor_2d(&a.xmap, false, static_cast<const int8_t*>(c.xq) + n0 * c.ldx, c.K, n,
                                  c.ldx, I8_KB, BN, true))
      return rc;
    a.xs = c.xs + n0;
    a.y = static_cast<Y*>(c.y) + n0 * c.ldy;
    a.N = (int)n;
    int cs = 1;
    if (int rc = split_of<BN, Y>(tiles * nt, a.nk, dev, &cs)) return rc;
    if (int rc = launch("k_int8_mm", k_int8_mm<BN, Y>, dim3(tiles * cs, (unsigned)nt), I8_THREADS, C::SMEM,
                        cs, st, a))
      return rc;
  }
  return OK;
}

template <typename Y>
int launch_pair(const Int8Call& c, I8Args& a, const DeviceInfo& dev, cudaStream_t st) {
  if (int rc = allow_max_smem((const void*)k_int8_pair<Y>, dev)) return rc;
  const int64_t mt = (c.M + 2 * I8_M - 1) / (2 * I8_M);
  const int64_t step = std::max<int64_t>(1, (((int64_t)1 << 30) / mt)) * 32;  // tiles of one launch below 2^30
  const int most = dev.sms / 2;
  for (int64_t n0 = 0; n0 < c.N; n0 += step) {
    const int64_t n = std::min(step, c.N - n0);
    // the tile width whose rounds over the pairs cost least: a tile's time is that
    // of its width and about 140 columns more (4096 tokens, 4096 -> 22016: 8.0 us
    // a round of 128 columns, 11.8 of 256; 1000 tokens, 2064 -> 5003: 80 tiles of
    // 256 in two rounds take 24 us, 120 of 192 in two 21)
    int width = PR_N;
    int64_t cost = -1;
    for (int w = PR_N; w >= 32; w -= 32) {
      const int64_t rounds = (mt * ((n + w - 1) / w) + most - 1) / most, cw = rounds * (w + 140);
      if (cost < 0 || cw < cost) {
        cost = cw;
        width = w;
      }
    }
    const int64_t ntn = (n + width - 1) / width;
    if (int rc = encode_tensor_2d(&a.wmap, false, c.wq, c.K, c.M, c.ldw, I8_KB, I8_M, true)) return rc;
    if (int rc = encode_tensor_2d(&a.xmap, false, static_cast<const int8_t*>(c.xq) + n0 * c.ldx, c.K, n,
                                  c.ldx, I8_KB, width / 2, true))
      return rc;
    a.xs = c.xs + n0;
    a.y = static_cast<Y*>(c.y) + n0 * c.ldy;
    a.N = (int)n;
    const int64_t tiles = mt * ntn;
    const int pairs = (int)std::min<int64_t>(tiles, most);
    // the cluster size is the kernel's own
    if (int rc = launch("k_int8_pair", k_int8_pair<Y>, dim3(2 * pairs), PR_THREADS, PR_SMEM, 0, st, a, width, (int)ntn,
                        (int)tiles))
      return rc;
  }
  return OK;
}

template <typename Y>
int matmul_as(const Int8Call& c, I8Args& a, const DeviceInfo& dev, cudaStream_t st) {
  if (c.N <= 16) return launch_mm<16, Y>(c, a, dev, st);
  if (c.N <= 32) return launch_mm<32, Y>(c, a, dev, st);
  if (c.N <= 64) return launch_mm<64, Y>(c, a, dev, st);
  // Up to 128 tokens single CTAs (100 tokens, 4096 -> 22016: 21 us against 24 in
  // pairs; 128 tokens, 4096 -> 4096: 9.7 and 12), above that pairs (129 tokens,
  // 4096 -> 11008: 17 and 13.5; 512 tokens 29 and 22), but for few tiles that a
  // cluster of 4 or more splits, with one CTA per SM (256 tokens, 4096 -> 1024: 8.2
  // and 11.0) or a deep product (256 tokens, 11008 -> 4096: 18.3 and 22.9; 4096 ->
  // 4096 12.1 and 11.6)
  if (c.N <= 128) return launch_mm<128, Y>(c, a, dev, st);
  const int64_t tiles = (c.M + I8_M - 1) / I8_M * ((c.N + 127) / 128);
  if (tiles * 4 <= dev.sms || (a.nk >= 64 && tiles * 2 <= dev.sms)) {
    int cs = 1;
    if (int rc = allow_max_smem((const void*)k_int8_mm<128, Y>, dev)) return rc;
    if (int rc = split_of<128, Y>(tiles, a.nk, dev, &cs)) return rc;
    if (cs >= 4) return launch_mm<128, Y>(c, a, dev, st);
  }
  return launch_pair<Y>(c, a, dev, st);
}

}  // namespace

namespace {
template <typename T>
int quantize_as(const T* x, int64_t ldx, int64_t N, int64_t K, int8_t* q, int64_t ldq, float* s, cudaStream_t st) {
  const bool vec = K % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0 &&
                   (N == 1 || (ldx * (int64_t)sizeof(T) % 16 == 0 && ldq % 8 == 0));
  constexpr int64_t kStep = (int64_t)1 << 30;  // rows of one launch
  for (int64_t n0 = 0; n0 < N; n0 += kStep) {
    const dim3 grid((unsigned)std::min(kStep, N - n0));
    if (int rc = launch("k_quant_rows", vec ? k_quant_rows<T, true> : k_quant_rows<T, false>, grid, RQ_THREADS, 0, 0,
                        st, x + n0 * ldx, ldx, (int)K, q + n0 * ldq, ldq, s + n0))
      return rc;
  }
  return OK;
}
}  // namespace

int int8_quantize(const void* x, int xdt, int64_t ldx, int64_t N, int64_t K, void* q, int64_t ldq, float* s,
                  cudaStream_t st) {
  int8_t* qq = static_cast<int8_t*>(q);
  if (xdt == 0) return quantize_as(static_cast<const float*>(x), ldx, N, K, qq, ldq, s, st);
  if (xdt == 1) return quantize_as(static_cast<const __nv_bfloat16*>(x), ldx, N, K, qq, ldq, s, st);
  return quantize_as(static_cast<const __half*>(x), ldx, N, K, qq, ldq, s, st);
}

int int8_matmul(const Int8Call& c, bool early_w, cudaStream_t st) {
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  I8Args a;
  memset(&a, 0, sizeof(a));
  a.ws = c.ws;
  a.bias = c.bias;
  a.ldy = c.ldy;
  a.M = (int)c.M;
  a.nk = (int)((c.K + I8_KB - 1) / I8_KB);
  a.early_w = early_w;
  if (c.ydt == 0) return matmul_as<float>(c, a, dev, st);
  if (c.ydt == 1) return matmul_as<__nv_bfloat16>(c, a, dev, st);
  return matmul_as<__half>(c, a, dev, st);
}

int set_i8_spin_limit(long long cycles) {
  const cudaError_t e = cudaMemcpyToSymbol(g_i8_spin_limit, &cycles, sizeof(cycles));
  if (e == cudaSuccess) return OK;
  return set_error(ERR_CUDA, "setting the wait limit: %s", cudaGetErrorString(e));
}

int read_i8_error(int clear, cudaStream_t st, int* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_i8_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess)
    return set_error(ERR_CUDA, "reading the device error word: %s", cudaGetErrorString(e));
  if (clear && v) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_i8_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess)
      return set_error(ERR_CUDA, "clearing the device error word: %s", cudaGetErrorString(e));
  }
  *out = v;
  return OK;
}

}  // namespace qg
