// int8 matrix products with one scale per token and one per channel:
//   y[n][m] = (sum_k xq[n][k] wq[m][k]) * xs[n] * ws[m] (+ bias[m])
// and the rounding of activations to int8 with one scale per row:
//   xs = max |x| / 127,  xq = rint(x / xs).
//
// The sum is exact: tcgen05.mma kind::i8 accumulates in int32, which holds
// K * 128 * 128 for K below 2^17 (larger K is refused).  It becomes fp32 once,
// is multiplied by the two scales in turn, the bias is added, and the result
// is rounded to y's type: four roundings of an fp32 ulp's half, then y's.
//
// Weights take the MMA's M side (128 channels per tile), tokens its N side,
// so that one kernel serves a single token (N = 16 columns, mostly idle: the
// weights' stream is what counts) and a long prompt (256 tokens per tile).
// Both operands are K-major int8 rows, copied by TMA as boxes of 128 bytes
// with 128-byte swizzle, the layout the tensor core reads; rows and columns
// past the end read as zeros.  A CTA has a producer warp, an MMA warp and four
// epilogue warps (one per TMEM lane quarter: lane = channel, column = token).
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

__device__ __forceinline__ int8_t quant1(float v, float s) {
  // IEEE division: the rounding of x / s is the definition's
  const float r = rintf(__fdiv_rn(v, s));
  return (int8_t)fminf(fmaxf(r, -127.0f), 127.0f);
}

constexpr int RQ_THREADS = 256;

// One CTA per row.  A row with a NaN or an infinity gets the scale NaN and
// zeros; an all-zero row (or one whose scale underflows to 0) the scale 0 and
// zeros.  Columns [K, kpad) get zeros.
template <typename T>
__global__ void __launch_bounds__(RQ_THREADS) k_quant_rows(const T* __restrict__ x, int64_t ldx, int K,
                                                           int8_t* __restrict__ q, int64_t ldq, int kpad,
                                                           float* __restrict__ s) {
  __shared__ uint32_t red[RQ_THREADS / 32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  int8_t* qr = q + row * ldq;
  uint32_t m = 0u;
  for (int k = threadIdx.x; k < K; k += RQ_THREADS) m = max(m, __float_as_uint(as_f32(xr[k])) & 0x7FFFFFFFu);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RQ_THREADS / 32; ++i) m = max(m, red[i]);
  const bool bad = m >= 0x7F800000u;
  const float sc = bad ? __int_as_float(0x7FC00000) : __fdiv_rn(__uint_as_float(m), 127.0f);
  for (int k = threadIdx.x; k < kpad; k += RQ_THREADS)
    qr[k] = k < K && sc > 0.0f ? quant1(as_f32(xr[k]), sc) : (int8_t)0;
  if (threadIdx.x == 0) s[row] = sc;
}

// ---------------------------------------------------------------- product
struct I8Args {
  alignas(64) CUtensorMap wmap;  // [M][K] int8, boxes of 128 bytes x 128 rows
  alignas(64) CUtensorMap xmap;  // [N][K] int8, boxes of 128 bytes x BN rows
  const float* xs;
  const float* ws;
  const float* bias;
  void* y;
  int64_t ldy;
  int ydt;
  int M, N, nk;    // nk: K steps
  int early_w;     // the weights may be read before the dependency wait
};

// BN tokens per tile; S ring stages.  kind::i8: s32 accumulators (bits 4-5 =
// 2), A and B signed (bits 7-9, 10-12 = 1), both K-major, N >> 3 at bit 17,
// M >> 4 at bit 24.
template <int BN>
struct I8Cfg {
  static constexpr int STAGE = I8_ABYTES + BN * I8_KB;
  static constexpr int S = BN == 256 ? 4 : BN == 128 ? 3 : 4;
  static constexpr int COLS = BN < 32 ? 32 : BN;  // TMEM columns
  static constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) |
                                    ((uint32_t)(I8_M >> 4) << 24);
  static constexpr size_t SMEM = (size_t)S * STAGE + 1024;
};

__device__ __forceinline__ void store_y(const I8Args& p, int64_t i, float v) {
  if (p.ydt == 0) static_cast<float*>(p.y)[i] = v;
  else if (p.ydt == 1) static_cast<__nv_bfloat16*>(p.y)[i] = __float2bfloat16(v);
  else static_cast<__half*>(p.y)[i] = __float2half(v);
}

// Grid (channel tiles x cluster size, token tiles).  The CTAs of a cluster
// split the K steps of one tile; their int32 parts are added through
// distributed shared memory (exact, so in any order).
template <int BN>
__global__ void __launch_bounds__(I8_THREADS) k_int8_mm(const __grid_constant__ I8Args p) {
  using C = I8Cfg<BN>;
  constexpr int S = C::S;
  extern __shared__ uint8_t i8_smem_raw[];
  __shared__ __align__(8) unsigned long long full[S], empty[S], done;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  cg::cluster_group cl = cg::this_cluster();
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

  if (warp == 0) {
    if (lane == 0) {
      const int pre = min(S, steps);
      auto load_w = [&](int i) {
        mbar_expect_tx(saddr(&full[i % S]), C::STAGE);
        tensor_g2s(ring_s + (i % S) * C::STAGE, &p.wmap, (k0 + i) * I8_KB, m0, saddr(&full[i % S]));
      };
      auto load_x = [&](int i) {
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
        if (!mbar_wait(saddr(&empty[i % S]), (uint32_t)((i / S - 1) & 1), &abort_flag)) break;
        load_w(i);
        load_x(i);
        issued = i + 1;
      }
      // no copy outlives the CTA, whatever the other warps gave up on
      for (int i = max(0, issued - S); i < issued; ++i)
        mbar_wait_drain(saddr(&full[i % S]), (uint32_t)((i / S) & 1));
    }
  } else if (warp == 1) {
    if (lane == 0) {
      pdl_wait();  // so that the bounded waits below do not count the previous kernel's time
      bool ok = true;
      for (int i = 0; i < steps && ok; ++i) {
        const int s = i % S;
        ok = mbar_wait(saddr(&full[s]), (uint32_t)((i / S) & 1), &abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint64_t da = sw128_desc(ring_s + s * C::STAGE),
                       db = sw128_desc(ring_s + s * C::STAGE + I8_ABYTES);
#pragma unroll
        for (int k = 0; k < I8_KB / 32; ++k)
          asm volatile(
              "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
              " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem),
              "l"(da + (uint64_t)(k * 2)), "l"(db + (uint64_t)(k * 2)), "r"(C::IDESC),
              "r"(i > 0 || k > 0 ? 1 : 0)
              : "memory");
        tc_commit(saddr(&empty[s]));
      }
      tc_commit(saddr(&done));
      mbar_wait_drain(saddr(&done), 0u);  // no MMA outlives its operands or the accumulators
    }
  } else {
    pdl_wait();  // xs
    if (warp == 2) pdl_trigger();
    mbar_wait(saddr(&done), 0u, &abort_flag);
    __syncwarp();
    tc_fence_after();
    const int quarter = warp & 3, row = quarter * 32 + lane, m = m0 + row;
    const float ws = m < p.M ? p.ws[m] : 0.0f, b = m < p.M && p.bias ? p.bias[m] : 0.0f;
    const uint32_t ta = tmem + ((uint32_t)(quarter * 32) << 16);
    int* part = reinterpret_cast<int*>(ring);  // [BN][128], once the ring is idle (done)
    const int nn = min(BN, p.N - n0);
    for (int c = 0; c < nn; c += 16) {
      uint32_t v[16];
      tmem_ld<16>(ta + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (cs > 1) {
          part[(c + j) * I8_M + row] = (int)v[j];
        } else if (c + j < nn && m < p.M) {
          const float f = (float)(int)v[j] * p.xs[n0 + c + j] * ws;
          store_y(p, (int64_t)(n0 + c + j) * p.ldy + m, p.bias ? f + b : f);
        }
      }
    }
  }
  __syncwarp();
  if (cs > 1) {
    cl.sync();
    if (warp >= 2) {
      int* part = reinterpret_cast<int*>(ring);
      const int row = (warp & 3) * 32 + lane, m = m0 + row, nn = min(BN, p.N - n0);
      if (m < p.M) {
        const float ws = p.ws[m], b = p.bias ? p.bias[m] : 0.0f;
        for (int c = rank; c < nn; c += cs) {
          int v = 0;
          for (int r = 0; r < cs; ++r) v += cl.map_shared_rank(part, r)[c * I8_M + row];
          const float f = (float)v * p.xs[n0 + c] * ws;
          store_y(p, (int64_t)(n0 + c) * p.ldy + m, p.bias ? f + b : f);
        }
      }
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
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, f, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  }
  return OK;
}

template <int BN>
int launch_mm(const Int8Call& c, I8Args& a, const DeviceInfo& dev, cudaStream_t st) {
  using C = I8Cfg<BN>;
  if (int rc = allow_max_smem((const void*)k_int8_mm<BN>, dev)) return rc;
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
    a.y = static_cast<uint8_t*>(c.y) + n0 * c.ldy * (c.ydt == 0 ? 4 : 2);
    a.N = (int)n;
    // few tiles: a cluster splits the K steps, as many CTAs as fit at once
    const int per_sm = std::max(1, (int)((size_t)dev.smem_optin / C::SMEM));
    int cs = 1;
    while (cs < 8 && tiles * nt * cs * 2 <= (int64_t)per_sm * dev.sms && a.nk >= cs * 4) cs *= 2;
    if (int rc = launch("k_int8_mm", k_int8_mm<BN>, dim3(tiles * cs, (unsigned)nt), I8_THREADS, C::SMEM,
                        cs, st, a))
      return rc;
  }
  return OK;
}

}  // namespace

int int8_quantize(const void* x, int xdt, int64_t ldx, int64_t N, int64_t K, void* q, int64_t ldq,
                  int64_t kpad, float* s, cudaStream_t st) {
  int8_t* qq = static_cast<int8_t*>(q);
  constexpr int64_t kStep = (int64_t)1 << 30;  // rows of one launch
  for (int64_t n0 = 0; n0 < N; n0 += kStep) {
    const dim3 grid((unsigned)std::min(kStep, N - n0));
    int rc;
    if (xdt == 0)
      rc = launch("k_quant_rows", k_quant_rows<float>, grid, RQ_THREADS, 0, 1, st,
                  static_cast<const float*>(x) + n0 * ldx, ldx, (int)K, qq + n0 * ldq, ldq, (int)kpad, s + n0);
    else if (xdt == 1)
      rc = launch("k_quant_rows", k_quant_rows<__nv_bfloat16>, grid, RQ_THREADS, 0, 1, st,
                  static_cast<const __nv_bfloat16*>(x) + n0 * ldx, ldx, (int)K, qq + n0 * ldq, ldq,
                  (int)kpad, s + n0);
    else
      rc = launch("k_quant_rows", k_quant_rows<__half>, grid, RQ_THREADS, 0, 1, st,
                  static_cast<const __half*>(x) + n0 * ldx, ldx, (int)K, qq + n0 * ldq, ldq, (int)kpad, s + n0);
    if (rc) return rc;
  }
  return OK;
}

int int8_matmul(const Int8Call& c, bool early_w, cudaStream_t st) {
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  I8Args a;
  memset(&a, 0, sizeof(a));
  a.ws = c.ws;
  a.bias = c.bias;
  a.ldy = c.ldy;
  a.ydt = c.ydt;
  a.M = (int)c.M;
  a.nk = (int)((c.K + I8_KB - 1) / I8_KB);
  a.early_w = early_w;
  if (c.N <= 16) return launch_mm<16>(c, a, dev, st);
  if (c.N <= 32) return launch_mm<32>(c, a, dev, st);
  if (c.N <= 64) return launch_mm<64>(c, a, dev, st);
  if (c.N <= 128) return launch_mm<128>(c, a, dev, st);
  return launch_mm<256>(c, a, dev, st);
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
