// Mixture-of-experts layer for a few tokens: router, SwiGLU experts in q8_0 /
// q4_0, and the weighted sum over each token's experts.
//
//   logits[n][e] = sum_k x[n][k] router[e][k]
//   ids[n][:], w[n][:] = the k best experts of token n and their weights
//   h[n][j] = w[n][j] silu(gate_e x_n) (up_e x_n),  e = ids[n][j]
//   y[n] = sum_j down_e h[n][j]
//
// Three launches, chained by programmatic dependent launch (no kernel waits on
// another's blocks, no counters, no atomics on global memory):
//
//  * k_moe_route: one cluster of 8 CTAs per 8 tokens; logits in 64-bit sums,
//    rounded to fp32 once (so the choice of experts does not depend on the
//    order of the sum), exchanged through distributed shared memory, then the
//    top k of each token by one warp.  Further CTAs of the same launch round x
//    to block fixed point (below).
//  * k_moe_up: work units of one expert x 32 h rows.  Each of a CTA's 4 warps
//    streams 8 gate rows and the same 8 up rows as one 16-row MMA tile, so
//    silu(gate) * up is lane-local; the unit's 32 h values of a token are one
//    block of the down projection, rounded to fixed point right there.
//  * k_moe_down: a CTA owns 64 rows of y (16 per warp); a cluster of CTAs
//    splits the chosen experts' columns and adds its parts through distributed
//    shared memory in rank order (deterministic).
//
// The arithmetic is the library's exact-integer scheme.  A block of 32
// activations is rounded to integers X = rint(x FX / max |x|), FX = 0x7F7F7F
// (a step of max |x| 2^-23; the GEMVs' powers of two leave 2^-22 to 2^-21, and
// here two products follow one another: measured 7.5e-7 -> 2.9e-7 relative
// error of y), and split into three signed byte digits
// X = p0 + 2^8 p1 + 2^16 p2; the integer dots of the block's quants with the
// digits are exact (mma.sync.m16n8k32.s8, |S| <= 32 * 128 * 128 = 2^19), and
// each block is scaled once: acc += (S0 + 2^8 S1 + 2^16 S2) (d max / FX).  With one or two
// tokens the three digits of both are the 8 columns of ONE MMA; with more,
// each digit plane has an MMA of 8 tokens.  The MMA's accumulator starts at
// the bits of 1.5 * 2^23, so that its integer result read as a float is
// 1.5 * 2^23 + S exactly: one subtraction instead of an integer conversion.
// A block that holds a NaN or an infinity gets a NaN scale: y is NaN there.
//
// Weights are "expert tiles", laid out once: per expert, 16-row tiles; a
// tile's groups of 128 columns are consecutive, each group the four blocks'
// quants in MMA fragment order (one 16-byte shared-memory load per lane is a
// q8_0 A fragment, or two of q4_0) and then the scales [8 rows][4 blocks][row,
// row + 8].  q4_0 nibbles are stored with bit 3 flipped: n ^ 8 shifted into
// the high half of a byte is 16 (n - 8) as a signed byte, one or two
// instructions; the 1/16 is folded into the activation scale (exact).  A warp
// reads its tile as one contiguous stream through a private cp.async ring.
#include <algorithm>

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "qgemv_common.cuh"
#include "qgemv_internal.h"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace qg {

namespace {

constexpr int MOE_NT = kMoeTokens;  // tokens per pass
constexpr int MOE_W = 4;            // warps per CTA of the expert kernels
constexpr int MOE_GCOLS = 128;      // columns of a group (4 blocks)
constexpr int MOE_DIG = 384;        // digit bytes of a group: [3 planes][4 lanes][32]
constexpr int MOE_ENT = 16;         // tokens of one entry, at most
constexpr float MOE_MAGIC = 12582912.0f;  // 1.5 * 2^23
constexpr uint32_t MOE_MAGIC_BITS = 0x4B400000u;

// bytes of a group (16 rows x 128 columns): quants, then 64 fp16 scales
template <int FMT> __host__ __device__ constexpr int grp_q() { return FMT == 8 ? 2048 : 1024; }
template <int FMT> __host__ __device__ constexpr int grp_bytes() { return grp_q<FMT>() + 128; }
// ring slots per warp: about 11 KB either way, 44 KB per CTA, 4 CTAs per SM
template <int FMT> __host__ __device__ constexpr int ring_depth() { return FMT == 8 ? 5 : 10; }

__host__ __device__ constexpr int groups_of(int64_t cols) {
  return (int)((cols + MOE_GCOLS - 1) / MOE_GCOLS);
}

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ float load_as_f32(const void* p, int dt, int64_t i) {
  if (dt == 0) return static_cast<const float*>(p)[i];
  if (dt == 1) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}

// ---------------------------------------------------------- fixed point
// The factors of a block from its largest |x| (as bits); every lane of the
// block gets the same.  X = rint(x up s), x = X * scale.
struct BlockScale {
  float up;     // 2^64 for blocks below 2^-64, so that s stays in range; else 1
  float s;      // FX / (max up); 0 for an all-zero or non-finite block (X = 0)
  float scale;  // max / FX; 0 for an all-zero block, NaN for a non-finite one
};
constexpr float MOE_FX = 8355711.0f;  // 0x7F7F7F: three signed byte digits of 127
__device__ __forceinline__ BlockScale block_scale(uint32_t amax) {
  BlockScale b{1.0f, 0.0f, 0.0f};
  const float m = __uint_as_float(amax);
  if (amax >= 0x7F800000u) {
    b.scale = __int_as_float(0x7FC00000);
  } else if (amax != 0u) {
    const bool tiny = m < 5.421010862427522e-20f;  // 2^-64
    b.up = tiny ? 18446744073709551616.0f : 1.0f;
    b.s = MOE_FX / (m * b.up);
    b.scale = m * b.up / MOE_FX * (tiny ? 5.421010862427522e-20f : 1.0f);
  }
  return b;
}
// X + 0x808080 of one value: byte p, with its top bit flipped, is digit p.
// |X| <= 0x7F7F7F also where the product rounds up (the clamp), so the biased
// value keeps to 24 bits.  A value of a non-finite block gives 0.
__device__ __forceinline__ uint32_t fixed_biased(float v, const BlockScale& b) {
  const int X = b.s == 0.0f ? 0 : __float2int_rn(v * b.up * b.s);
  return (uint32_t)(min(max(X, -0x7F7F7F), 0x7F7F7F) + 0x808080);
}

struct MoeArgs {
  // activations and their fixed-point form
  const void* x;
  int64_t ldx;
  int xdt;
  uint8_t* xdig;   // [N][K groups][384]
  float* xs;       // [N][K groups * 4]
  uint8_t* hdig;   // [N * slots][F groups][384]
  float* hs;       // [N * slots][F groups * 4]
  // choices
  const int* ids;        // [N][slots]
  const float* weights;  // [N][slots]
  int N, slots;
  // experts
  const uint8_t* gate_up;
  const uint8_t* down;
  int E, K, F;     // E counts the shared experts too
  int max_ent;
  // output
  void* y;
  int64_t ldy;
};

struct RouteArgs {
  const void* w;   // router [E][K]
  int wdt;
  int64_t ldw;
  const float* bias;
  int E, K, k, scoring, normalize, shared;
  float scale;
  int* ids;        // [N][k + shared]
  float* weights;
  int clusters;    // CTAs [0, 8 * clusters) route; the others prepare x
};

// Fixed-point form of x, one warp per (token, group of 128 columns); columns
// past K get zero digits and a zero scale.  Also the zero scales of h's blocks
// past F (their digits are never read into a nonzero product, but a stale NaN
// scale would be).
__device__ void prepare_x(const MoeArgs& a, int warp, int nwarps, int lane) {
  const int kg = groups_of(a.K), fg = groups_of(a.F), fb = a.F / QK;
  for (int i = warp; i < a.N * kg; i += nwarps) {
    const int n = i / kg, g = i % kg;
    const int k0 = g * MOE_GCOLS + lane * 4;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (k0 < a.K)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = load_as_f32(a.x, a.xdt, (int64_t)n * a.ldx + k0 + j);
    uint32_t m = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const BlockScale b = block_scale(m);
    uint32_t f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = fixed_biased(v[j], b);
    // lane 8 blk + j holds elements 4j ... of block blk: B fragment register
    // j / 4 of MMA lane j % 4
    const int blk = lane >> 3, t = lane & 3, half = (lane >> 2) & 1;
    uint8_t* dst = a.xdig + (int64_t)i * MOE_DIG + t * 32 + blk * 8 + half * 4;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t w = ((f[0] >> (8 * p)) & 0xFFu) | (((f[1] >> (8 * p)) & 0xFFu) << 8) |
                         (((f[2] >> (8 * p)) & 0xFFu) << 16) | (((f[3] >> (8 * p)) & 0xFFu) << 24);
      *reinterpret_cast<uint32_t*>(dst + p * 128) = w ^ 0x80808080u;
    }
    if ((lane & 7) == 0) a.xs[(int64_t)i * 4 + blk] = b.scale;
  }
  const int pad = fg * 4 - fb;
  for (int i = warp * 32 + lane; i < a.N * a.slots * pad; i += nwarps * 32)
    a.hs[(int64_t)(i / pad) * fg * 4 + fb + i % pad] = 0.0f;
}

// ------------------------------------------------------------- routing
constexpr int RT_THREADS = 256;
constexpr int RT_WARPS = RT_THREADS / 32;
constexpr int RT_CL = 8;    // CTAs of a routing cluster
constexpr int RT_TE = 4;    // experts of a warp's tile
// x columns staged at a time, as doubles (32 KB)
template <int TN> __host__ __device__ constexpr int rt_chunk() { return TN == 1 ? 4096 : 512; }

// Ordering key of a score: larger key = larger score; NaN lowest; +0 == -0.
__device__ __forceinline__ unsigned long long rank_key(double v) {
  if (v != v) return 0ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ double load_as_f64(const void* p, int dt, int64_t i) {
  return (double)load_as_f32(p, dt, i);
}

// Four consecutive values from element i on as fp32, those past `n` zero; one
// load where `vec` says that i % 4 == 0 starts an aligned one.
__device__ __forceinline__ void load4(float (&v)[4], const void* p, int dt, int64_t i, int n, bool vec) {
  if (vec && n >= 4) {
    if (dt == 0) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      v[0] = f.x;
      v[1] = f.y;
      v[2] = f.z;
      v[3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
      const uint32_t h[4] = {u.x & 0xFFFFu, u.x >> 16, u.y & 0xFFFFu, u.y >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = dt == 1 ? __uint_as_float(h[j] << 16) : __half2float(__ushort_as_half((unsigned short)h[j]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? load_as_f32(p, dt, i + j) : 0.0f;
  }
}

// The top k of one token by one warp: `logit` and `key` hold E values in
// shared memory.  Ties go to the lowest index.
__device__ void route_token(const RouteArgs& r, const float* logit, unsigned long long* key,
                            int n, int lane) {
  const int E = r.E;
  // statistics in 32 bits: max, sum of exp over all experts, any NaN
  float mx = -INFINITY;
  bool nan = false;
  for (int e = lane; e < E; e += 32) {
    mx = fmaxf(mx, logit[e]);
    nan |= logit[e] != logit[e];
  }
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  nan = __any_sync(0xffffffffu, nan);
  float all = 0.0f;
  double all64 = 0.0;
  if (r.scoring == 0) {
    for (int e = lane; e < E; e += 32) all += expf(logit[e] - mx);
    all = warp_sum(all);
    if (r.bias) {
      for (int e = lane; e < E; e += 32) all64 += exp((double)logit[e] - (double)mx);
      for (int o = 16; o; o >>= 1) all64 += __shfl_xor_sync(0xffffffffu, all64, o);
    }
  }
  // softmax and sigmoid are increasing, so without a bias the logits rank the
  // experts; with one the scores are formed in 64 bits, so that rounding does
  // not decide between near scores
  for (int e = lane; e < E; e += 32) {
    double v = (double)logit[e];
    if (r.bias)
      v = (r.scoring == 0 ? exp(v - (double)mx) / all64 : 1.0 / (1.0 + exp(-v))) + (double)r.bias[e];
    key[e] = rank_key(v);
  }
  __syncwarp();
  // each lane's best of its own experts (e = lane, lane + 32, ...); after a
  // round only the winner's lane looks again.  A taken expert is marked by
  // its bit (experts of a lane: at most 32).
  uint32_t taken = 0u;
  unsigned long long best = 0ull;
  int at = -1;
  auto look = [&]() {
    at = -1;
    best = 0ull;
    for (int i = 0, e = lane; e < E; ++i, e += 32)
      if (!((taken >> i) & 1u) && (at < 0 || key[e] > best)) {
        best = key[e];
        at = e;
      }
  };
  look();
  const int slots = r.k + r.shared;
  int mine = -1;  // lane j keeps the j-th choice
  for (int j = 0; j < r.k; ++j) {
    const uint32_t hi = at < 0 ? 0u : (uint32_t)(best >> 32), lo = at < 0 ? 0u : (uint32_t)best;
    const uint32_t mh = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t ml = __reduce_max_sync(0xffffffffu, hi == mh ? lo : 0u);
    const int win = (int)__reduce_min_sync(
        0xffffffffu, at >= 0 && hi == mh && lo == ml ? (uint32_t)at : 0xFFFFFFFFu);
    if (lane == j) mine = win;
    if (win == at) {
      taken |= 1u << (win >> 5);
      look();
    }
  }
  float s = 0.0f;
  if (lane < r.k) {
    const float l = logit[mine];
    s = r.scoring == 0 ? expf(l - mx) : 1.0f / (1.0f + expf(-l));
  }
  const float sum = warp_sum(s);
  if (lane < r.k) {
    // a sum below the smallest normal number (every chosen score underflowed)
    // divides as that number: weights of zero, not NaN
    const float den = r.normalize ? fmaxf(sum, 1.17549435e-38f) : r.scoring == 0 ? all : 1.0f;
    float w = s / den * r.scale;
    if (nan || sum != sum) w = __int_as_float(0x7FC00000);
    r.ids[(int64_t)n * slots + lane] = mine;
    r.weights[(int64_t)n * slots + lane] = w;
  } else if (lane < slots) {
    r.ids[(int64_t)n * slots + lane] = E + lane - r.k;
    r.weights[(int64_t)n * slots + lane] = 1.0f;
  }
}

// CTAs [0, 8 * clusters): cluster c routes tokens [TN c, TN c + TN), CTA rank
// r computing the logits of experts [E r / 8, E (r + 1) / 8) and choosing for
// token TN c + r.  A warp takes tiles of 4 experts x TN tokens; with fewer
// tiles than warps the columns are split over them too.  The sums are in
// fp64 (measured here: 64 FMA per clock and SM, the conversions from fp32 a
// quarter of that, which is why x is converted once per CTA).
template <int TN>
__global__ void __launch_bounds__(RT_THREADS, 2) k_moe_route(MoeArgs a, RouteArgs r) {
  extern __shared__ __align__(16) uint8_t rt_smem[];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((int)blockIdx.x >= RT_CL * r.clusters) {
    pdl_wait();
    prepare_x(a, (blockIdx.x - RT_CL * r.clusters) * RT_WARPS + warp,
              (gridDim.x - RT_CL * r.clusters) * RT_WARPS, lane);
    return;
  }
  constexpr int CH = rt_chunk<TN>();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), E = r.E, K = r.K;
  const int n0 = (blockIdx.x / RT_CL) * TN, nn = min(TN, a.N - n0);
  const int e0 = (int)((int64_t)E * rank / RT_CL), e1 = (int)((int64_t)E * (rank + 1) / RT_CL);
  const int ne = e1 - e0, epad = (E + RT_CL - 1) / RT_CL;
  // shared memory: x chunk [TN][CH] doubles, partial sums [8][epad][TN]
  // doubles, keys [E], this CTA's token's logits [E]
  double* xd = reinterpret_cast<double*>(rt_smem);
  double* part = xd + TN * CH;
  unsigned long long* key = reinterpret_cast<unsigned long long*>(part + RT_WARPS * epad * TN);
  float* logit = reinterpret_cast<float*>(key + E);
  const int tiles = (ne + RT_TE - 1) / RT_TE;
  int ks = 1;  // warps that share a tile's columns
  while (ks < RT_WARPS && ks * 2 * tiles <= RT_WARPS) ks *= 2;
  const int sl = warp % ks;
  pdl_wait();
  const bool vec = r.ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(r.w) & 15) == 0;
  for (int t0 = 0; t0 < tiles; t0 += RT_WARPS / ks) {
    const int tl = t0 + warp / ks, eb = e0 + tl * RT_TE;
    double acc[RT_TE * TN] = {};
    for (int c0 = 0; c0 < K; c0 += CH) {
      const int cn = min(CH, K - c0);
      __syncthreads();
      // column 128 i + 4 l + j sits at 128 i + 64 (j / 2) + 2 l + j % 2: a lane
      // reads its four columns with two conflict-free 16-byte loads
      for (int i = threadIdx.x; i < TN * CH; i += RT_THREADS) {
        const int n = i / CH, c = i % CH;
        const double v = n < nn && c < cn ? load_as_f64(a.x, a.xdt, (int64_t)(n0 + n) * a.ldx + c0 + c) : 0.0;
        xd[n * CH + (c & ~127) + ((c >> 1) & 1) * 64 + ((c >> 2) & 31) * 2 + (c & 1)] = v;
      }
      __syncthreads();
      if (tl < tiles) {
#pragma unroll 2
        for (int cb = sl * 128; cb < cn; cb += ks * 128) {
          float w[RT_TE][4];
#pragma unroll
          for (int i = 0; i < RT_TE; ++i)
            load4(w[i], r.w, r.wdt, (int64_t)min(eb + i, e1 - 1) * r.ldw + c0 + cb + 4 * lane,
                  cn - cb - 4 * lane, vec);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            double wd[RT_TE][2];
#pragma unroll
            for (int i = 0; i < RT_TE; ++i) {
              wd[i][0] = (double)w[i][2 * h];
              wd[i][1] = (double)w[i][2 * h + 1];
            }
#pragma unroll
            for (int n = 0; n < TN; ++n) {
              const double2 xv = *reinterpret_cast<const double2*>(xd + n * CH + cb + h * 64 + lane * 2);
#pragma unroll
              for (int i = 0; i < RT_TE; ++i) {
                acc[i * TN + n] = fma(wd[i][0], xv.x, acc[i * TN + n]);
                acc[i * TN + n] = fma(wd[i][1], xv.y, acc[i * TN + n]);
              }
            }
          }
        }
      }
    }
    if (tl < tiles) {
      // transposing butterfly: each step halves the values a lane holds
      constexpr int V = RT_TE * TN;
      int at = 0;
#pragma unroll
      for (int v = V / 2, o = 16; v >= 1; v /= 2, o /= 2) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < v; ++i) {
          const double give = up ? acc[i] : acc[i + v], keep = up ? acc[i + v] : acc[i];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
        at += up ? v : 0;
      }
      for (int o = 16 / V; o >= 1; o /= 2) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
      const int e = eb + at / TN - e0;
      if ((lane & (32 / V - 1)) == 0 && e < ne) part[(sl * epad + e) * TN + at % TN] = acc[0];
    }
  }
  cl.sync();  // every CTA of the cluster runs, and every partial sum is there
  for (int i = threadIdx.x; i < ne * nn; i += RT_THREADS) {
    const int e = i / nn, n = i % nn;
    double v = 0.0;
    for (int s = 0; s < ks; ++s) v += part[(s * epad + e) * TN + n];
    float* dst = cl.map_shared_rank(logit, n);  // CTA n chooses for token n
    dst[e0 + e] = (float)v;
  }
  cl.sync();
  if (warp == 0 && rank < nn) route_token(r, logit, key, n0 + rank, lane);
}

// --------------------------------------------------- entries of the experts
// The chosen experts in ascending order, each with up to 16 of its tokens (an
// expert with more has several entries), built by every CTA for itself from
// the choices.  A choice outside [0, E) selects nothing; an expert that one
// token names twice counts once, with the sum of the weights.  An expert's
// tokens are kept as a 64-bit mask and taken in ascending order: every CTA
// builds the same entries, since the CTAs share them out.
struct Table {
  uint32_t* mask;   // [E][2] tokens of the expert
  int* first;       // [E]
  uint32_t* ent;    // [max_ent] expert | first << 10 | count << 22
  uint32_t* tmp;    // [P]
  uint32_t* sorted; // [P] choice | token << 16, by expert
  float* w;         // [P]
  int nent;
};
__host__ __device__ __forceinline__ size_t table_bytes(int E, int P, int max_ent) {
  return (size_t)(3 * E + max_ent + 3 * P) * 4;
}

__device__ Table build_table(uint8_t* mem, const MoeArgs& a) {
  __shared__ uint32_t wsum[MOE_W];
  const int P = a.N * a.slots, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Table t;
  t.mask = reinterpret_cast<uint32_t*>(mem);
  t.first = reinterpret_cast<int*>(t.mask + 2 * a.E);
  t.ent = reinterpret_cast<uint32_t*>(t.first + a.E);
  t.tmp = t.ent + a.max_ent;
  t.sorted = t.tmp + P;
  t.w = reinterpret_cast<float*>(t.sorted + P);
  for (int i = tid; i < 2 * a.E; i += blockDim.x) t.mask[i] = 0u;
  for (int i = tid; i < P; i += blockDim.x) {
    t.sorted[i] = (uint32_t)a.ids[i];
    t.w[i] = a.weights[i];
  }
  __syncthreads();
  for (int p = tid; p < P; p += blockDim.x) {
    const uint32_t id = t.sorted[p];
    const int first = p / a.slots * a.slots;
    bool keep = id < (uint32_t)a.E;
    for (int q = first; q < p; ++q) keep &= t.sorted[q] != id;
    uint32_t v = 0xFFFFFFFFu;
    if (keep) {
      float w = t.w[p];
      for (int q = p + 1; q < first + a.slots; ++q)
        if (t.sorted[q] == id) w += t.w[q];  // a later duplicate's own entry is not written
      t.w[p] = w;
      const int n = p / a.slots;
      atomicOr(&t.mask[2 * id + (n >> 5)], 1u << (n & 31));
      v = id;
    }
    t.tmp[p] = v;
  }
  __syncthreads();
  // exclusive prefix sums of the counts (low half) and the entries (high half)
  const int per = (a.E + (int)blockDim.x - 1) / (int)blockDim.x;
  const int b = min(a.E, tid * per), e = min(a.E, b + per);
  auto count = [&](int i) { return (uint32_t)(__popc(t.mask[2 * i]) + __popc(t.mask[2 * i + 1])); };
  uint32_t sum = 0u;
  for (int i = b; i < e; ++i) {
    const uint32_t c = count(i);
    sum += c + ((c + MOE_ENT - 1) / MOE_ENT << 16);
  }
  uint32_t inc = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  uint32_t before = inc - sum, total = 0u;
  for (int i = 0; i < MOE_W; ++i) {
    if (i < warp) before += wsum[i];
    total += wsum[i];
  }
  uint32_t c0 = before & 0xFFFFu, n0 = before >> 16;
  for (int i = b; i < e; ++i) {
    const uint32_t c = count(i);
    for (uint32_t j = 0; j < c; j += MOE_ENT)
      t.ent[n0++] = (uint32_t)i | (c0 + j) << 10 | min((uint32_t)MOE_ENT, c - j) << 22;
    t.first[i] = (int)c0;
    c0 += c;
  }
  __syncthreads();
  for (int p = tid; p < P; p += blockDim.x) {
    const uint32_t id = t.tmp[p];
    if (id != 0xFFFFFFFFu) {
      const int n = p / a.slots;
      const uint32_t lo = t.mask[2 * id], hi = t.mask[2 * id + 1], below = (1u << (n & 31)) - 1u;
      const int rank = n < 32 ? __popc(lo & below) : __popc(lo) + __popc(hi & below);
      t.sorted[t.first[id] + rank] = (uint32_t)p | (uint32_t)n << 16;
    }
  }
  __syncthreads();
  t.nent = (int)(total >> 16);
  return t;
}

// ------------------------------------------------------- streaming products
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
// the previous kernel of the chain wrote these: coherent loads
__device__ __forceinline__ uint4 ldg128(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ void mma_s8(float (&f)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  uint32_t c[4];
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(MOE_MAGIC_BITS));
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(c[i]) - MOE_MAGIC;
}

// One warp's ring over a contiguous stream of groups.
template <int FMT>
struct Ring {
  uint32_t base;  // shared address of the warp's slots
  int in, out;    // next slot to fill / to read
  __device__ __forceinline__ void fill(const uint8_t* src, int lane) {
    constexpr int GB = grp_bytes<FMT>();
    const uint32_t dst = base + (uint32_t)(in * GB);
#pragma unroll
    for (int i = 0; i < grp_q<FMT>() / 512; ++i)
      cp16(dst + i * 512 + lane * 16, src + i * 512 + lane * 16);
    if (lane < 8) cp16(dst + grp_q<FMT>() + lane * 16, src + grp_q<FMT>() + lane * 16);
    in = in + 1 == ring_depth<FMT>() ? 0 : in + 1;
  }
};

// A fragments of blocks 2 * pr and 2 * pr + 1 of the group at `st`.
template <int FMT>
__device__ __forceinline__ void load_a(uint32_t (&a)[2][4], uint32_t st, int pr, int lane) {
  if (FMT == 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint4 v = lds128(st + (2 * pr + i) * 512 + lane * 16);
      a[i][0] = v.x;
      a[i][1] = v.y;
      a[i][2] = v.z;
      a[i][3] = v.w;
    }
  } else {
    // words: block 2 pr (row g, row g + 8), block 2 pr + 1 (row g, row g + 8)
    const uint4 v = lds128(st + pr * 512 + lane * 16);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        a[i][h] = (w[2 * i + h] << 4) & 0xF0F0F0F0u;      // columns 4t ...
        a[i][2 + h] = w[2 * i + h] & 0xF0F0F0F0u;         // columns 16 + 4t ...
      }
  }
}

// acc over the tokens of an entry: MODE 2 (one or two tokens, their digits the
// 8 columns of one MMA; acc[0], acc[1]: rows g and g + 8, this lane's digit
// pair), 8 (acc[0..1] row g, [2..3] row g + 8, tokens 2t and 2t + 1) or 16
// (then tokens 8 + 2t and 9 + 2t in acc[4..7]).
template <int MODE> __host__ __device__ constexpr int acc_n() { return MODE == 2 ? 2 : MODE / 2; }

// What an entry's tokens look like to a lane.
template <int FMT, int MODE>
struct Cols {
  const uint8_t* dig[MODE == 16 ? 2 : 1];  // this lane's digits (column lane / 4)
  const float* s[MODE == 2 ? 1 : MODE == 8 ? 2 : 4];  // scales of the lane's columns
  float f;  // MODE 2: weight of the lane's digit pair
  // row(i): the activation row of the entry's i-th token
  template <typename Row>
  __device__ __forceinline__ void set(const uint8_t* digits, const float* scales, int groups,
                                      int cnt, int lane, Row row) {
    const int n = lane >> 2, t = lane & 3;
    const int64_t ds = (int64_t)groups * MOE_DIG, ss = (int64_t)groups * 4;
    constexpr float Q = FMT == 8 ? 1.0f : 0.0625f;  // q4_0 quants come as 16 (n - 8)
    if (MODE == 2) {
      dig[0] = digits + row(min(n >> 2, cnt - 1)) * ds + (n & 3) * 128 + t * 32;
      s[0] = scales + row(min(t >> 1, cnt - 1)) * ss;
      f = ((t & 1) ? 65536.0f : 1.0f) * Q;
    } else {
      f = Q;
#pragma unroll
      for (int h = 0; h < MODE / 8; ++h) {
        dig[h] = digits + row(min(8 * h + n, cnt - 1)) * ds + t * 32;
        s[2 * h] = scales + row(min(8 * h + 2 * t, cnt - 1)) * ss;
        s[2 * h + 1] = scales + row(min(8 * h + 2 * t + 1, cnt - 1)) * ss;
      }
    }
  }
};

// One group: digits and scales of the columns (L1 / L2), then the quants.
template <int FMT, int MODE, typename Wait>
__device__ __forceinline__ void group_product(float (&acc)[acc_n<MODE>()], const Cols<FMT, MODE>& c,
                                              int grp, uint32_t st, int lane, Wait wait) {
  const uint32_t dst = st + grp_q<FMT>() + (lane >> 2) * 16;
  if constexpr (MODE == 2) {
    uint4 b[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (((lane >> 2) & 3) != 3) {
      b[0] = ldg128(c.dig[0] + grp * MOE_DIG);
      b[1] = ldg128(c.dig[0] + grp * MOE_DIG + 16);
    }
    const uint4 sv = ldg128(c.s[0] + grp * 4);
    wait();
    const uint4 dv = lds128(dst);
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      uint32_t a[2][4];
      load_a<FMT>(a, st, pr, lane);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[4];
        mma_s8(v, a[i], i ? b[pr].z : b[pr].x, i ? b[pr].w : b[pr].y);
        const int k = 2 * pr + i;
        const float sc = __uint_as_float(k == 0 ? sv.x : k == 1 ? sv.y : k == 2 ? sv.z : sv.w) * c.f;
        const uint32_t dw = k == 0 ? dv.x : k == 1 ? dv.y : k == 2 ? dv.z : dv.w;
        const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&dw));
        acc[0] = fmaf(fmaf(v[1], 256.0f, v[0]), d.x * sc, acc[0]);
        acc[1] = fmaf(fmaf(v[3], 256.0f, v[2]), d.y * sc, acc[1]);
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < MODE / 8; ++h) {
      uint4 b[3][2];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        b[p][0] = ldg128(c.dig[h] + grp * MOE_DIG + p * 128);
        b[p][1] = ldg128(c.dig[h] + grp * MOE_DIG + p * 128 + 16);
      }
      const uint4 s0 = ldg128(c.s[2 * h] + grp * 4), s1 = ldg128(c.s[2 * h + 1] + grp * 4);
      if (h == 0) wait();
      const uint4 dv = lds128(dst);
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        uint32_t a[2][4];
        load_a<FMT>(a, st, pr, lane);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v0[4], v1[4], v2[4];
          mma_s8(v0, a[i], i ? b[0][pr].z : b[0][pr].x, i ? b[0][pr].w : b[0][pr].y);
          mma_s8(v1, a[i], i ? b[1][pr].z : b[1][pr].x, i ? b[1][pr].w : b[1][pr].y);
          mma_s8(v2, a[i], i ? b[2][pr].z : b[2][pr].x, i ? b[2][pr].w : b[2][pr].y);
          const int k = 2 * pr + i;
          const float c0 = __uint_as_float(k == 0 ? s0.x : k == 1 ? s0.y : k == 2 ? s0.z : s0.w) * c.f;
          const float c1 = __uint_as_float(k == 0 ? s1.x : k == 1 ? s1.y : k == 2 ? s1.z : s1.w) * c.f;
          const uint32_t dw = k == 0 ? dv.x : k == 1 ? dv.y : k == 2 ? dv.z : dv.w;
          const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&dw));
          const float sc[4] = {d.x * c0, d.x * c1, d.y * c0, d.y * c1};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[4 * h + j] = fmaf(fmaf(v2[j], 65536.0f, fmaf(v1[j], 256.0f, v0[j])), sc[j],
                                  acc[4 * h + j]);
        }
      }
    }
  }
}

// The digit pairs of MODE 2 live in neighbouring lanes: their sum.
template <int MODE>
__device__ __forceinline__ void join(float (&acc)[acc_n<MODE>()]) {
  if constexpr (MODE == 2) {
    acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 1);
    acc[1] += __shfl_xor_sync(0xffffffffu, acc[1], 1);
  }
}

// f(token of the entry, first row value, second row value) for every column
// that this lane holds after join().
template <int MODE, typename F>
__device__ __forceinline__ void each_col(const float (&acc)[acc_n<MODE>()], int cnt, int lane, F f) {
  const int t = lane & 3;
  if constexpr (MODE == 2) {
    if (!(t & 1) && (t >> 1) < cnt) f(t >> 1, acc[0], acc[1]);
  } else {
#pragma unroll
    for (int h = 0; h < MODE / 8; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (8 * h + 2 * t + j < cnt) f(8 * h + 2 * t + j, acc[4 * h + j], acc[4 * h + 2 + j]);
  }
}

// ------------------------------------------------------------- gate and up
template <int FMT>
__global__ void __launch_bounds__(32 * MOE_W, 4) k_moe_up(MoeArgs a) {
  extern __shared__ __align__(128) uint8_t up_smem[];
  __shared__ float hbuf[2][MOE_ENT][32];
  constexpr int GB = grp_bytes<FMT>(), D = ring_depth<FMT>();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const Table tb = build_table(up_smem + (size_t)MOE_W * D * GB, a);
  const int fc = a.F / 32, kg = groups_of(a.K), fg = groups_of(a.F);
  const int units = tb.nent * fc;
  const int64_t tile = (int64_t)kg * GB;  // one 16-row tile
  Ring<FMT> ring{saddr(up_smem) + (uint32_t)(warp * D * GB), 0, 0};
  // the tile of unit u that this warp reads: expert, then 8-row pairs
  auto src_of = [&](int u) {
    const uint32_t en = tb.ent[u / fc];
    return a.gate_up + ((int64_t)(en & 1023u) * (a.F / 8) + (u % fc) * MOE_W + warp) * tile;
  };
  int pu = blockIdx.x, pg = 0;  // next group to ask for
  const uint8_t* psrc = pu < units ? src_of(pu) : nullptr;
  auto ask = [&]() {
    if (pu < units) {
      ring.fill(psrc + (int64_t)pg * GB, lane);
      if (++pg == kg) {
        pg = 0;
        pu += gridDim.x;
        if (pu < units) psrc = src_of(pu);
      }
    }
    cp_commit();
  };
  for (int i = 0; i < D; ++i) ask();
  int buf = 0;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const uint32_t en = tb.ent[u / fc];
    const int first = (en >> 10) & 0xFFF, cnt = en >> 22;
    auto run = [&](auto mode) {
      constexpr int MODE = decltype(mode)::value;
      float acc[acc_n<MODE>()] = {};
      Cols<FMT, MODE> cols;
      cols.set(a.xdig, a.xs, kg, cnt, lane,
               [&](int i) { return (int64_t)(tb.sorted[first + i] >> 16); });
      for (int g = 0; g < kg; ++g) {
        group_product<FMT, MODE>(acc, cols, g, ring.base + (uint32_t)(ring.out * GB), lane, [&]() {
          cp_wait<D - 1>();
          __syncwarp();
        });
        __syncwarp();  // every lane has read the slot
        ring.out = ring.out + 1 == D ? 0 : ring.out + 1;
        ask();
      }
      join<MODE>(acc);
      each_col<MODE>(acc, cnt, lane, [&](int i, float gate, float up) {
        const float w = tb.w[tb.sorted[first + i] & 0xFFFFu];
        hbuf[buf][i][warp * 8 + (lane >> 2)] = gate / (1.0f + expf(-gate)) * up * w;
      });
    };
    if (cnt <= 2) run(std::integral_constant<int, 2>());
    else if (cnt <= 8) run(std::integral_constant<int, 8>());
    else run(std::integral_constant<int, 16>());
    __syncthreads();
    // the unit's 32 values of a token are block u % fc of its h
    const int hb = u % fc;
    for (int i = warp; i < cnt; i += MOE_W) {
      const float v = hbuf[buf][i][lane];
      const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7FFFFFFFu);
      const BlockScale b = block_scale(m);
      const uint32_t f = fixed_biased(v, b) ^ 0x808080u;
      const int64_t row = tb.sorted[first + i] & 0xFFFFu;
      uint8_t* dst = a.hdig + (row * fg + (hb >> 2)) * MOE_DIG + ((lane >> 2) & 3) * 32 +
                     (hb & 3) * 8 + (lane >> 4) * 4 + (lane & 3);
#pragma unroll
      for (int p = 0; p < 3; ++p) dst[p * 128] = (uint8_t)(f >> (8 * p));
      if (lane == 0) a.hs[row * fg * 4 + hb] = b.scale;
    }
    buf ^= 1;  // the next unit's values go to the other buffer, so one barrier a unit is enough
  }
}

// -------------------------------------------------------------------- down
template <int FMT>
__global__ void __launch_bounds__(32 * MOE_W, 4) k_moe_down(MoeArgs a, int ydt) {
  extern __shared__ __align__(128) uint8_t dn_smem[];
  constexpr int GB = grp_bytes<FMT>(), D = ring_depth<FMT>();
  cg::cluster_group cl = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  // the choices were complete before k_moe_up passed its own wait and
  // allowed this launch; what k_moe_up writes comes after the wait below
  const size_t yb = (size_t)a.N * 16 * MOE_W * 4;
  float* ypart = reinterpret_cast<float*>(dn_smem + (size_t)MOE_W * D * GB);
  const Table tb = build_table(dn_smem + (size_t)MOE_W * D * GB + yb, a);
  const int fg = groups_of(a.F);
  const int64_t total = (int64_t)tb.nent * fg;
  const int q0 = (int)(total * rank / cs), q1 = (int)(total * (rank + 1) / cs);
  const int rt = blockIdx.x / cs * MOE_W + warp, nrt = a.K / 16;  // this warp's 16 rows
  const bool live = rt < nrt;
  const int64_t tile = (int64_t)fg * GB;
  Ring<FMT> ring{saddr(dn_smem) + (uint32_t)(warp * D * GB), 0, 0};
  auto src_of = [&](int en) {
    return a.down + ((int64_t)(tb.ent[en] & 1023u) * nrt + rt) * tile;
  };
  int pq = q0, pe = q0 / fg, pg = q0 % fg;
  const uint8_t* psrc = live && q0 < q1 ? src_of(pe) : nullptr;
  auto ask = [&]() {
    if (live && pq < q1) {
      ring.fill(psrc + (int64_t)pg * GB, lane);
      ++pq;
      if (++pg == fg) {
        pg = 0;
        ++pe;
        if (pq < q1) psrc = src_of(pe);
      }
    }
    cp_commit();
  };
  for (int i = 0; i < D; ++i) ask();
  for (int i = threadIdx.x; i < a.N * 16 * MOE_W; i += 32 * MOE_W) ypart[i] = 0.0f;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  if (live) {
    for (int q = q0; q < q1;) {
      const int e = q / fg, g0 = q % fg, g1 = min(fg, g0 + q1 - q);
      const uint32_t en = tb.ent[e];
      const int first = (en >> 10) & 0xFFF, cnt = en >> 22;
      auto run = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        float acc[acc_n<MODE>()] = {};
        Cols<FMT, MODE> cols;
        cols.set(a.hdig, a.hs, fg, cnt, lane,
                 [&](int i) { return (int64_t)(tb.sorted[first + i] & 0xFFFFu); });
        for (int g = g0; g < g1; ++g) {
          group_product<FMT, MODE>(acc, cols, g, ring.base + (uint32_t)(ring.out * GB), lane, [&]() {
            cp_wait<D - 1>();
            __syncwarp();
          });
          __syncwarp();
          ring.out = ring.out + 1 == D ? 0 : ring.out + 1;
          ask();
        }
        join<MODE>(acc);
        // tokens of an entry are distinct, and the rows are this warp's own
        each_col<MODE>(acc, cnt, lane, [&](int i, float lo, float hi) {
          float* p = ypart + (tb.sorted[first + i] >> 16) * 16 * MOE_W + warp * 16 + (lane >> 2);
          p[0] += lo;
          p[8] += hi;
        });
      };
      if (cnt <= 2) run(std::integral_constant<int, 2>());
      else if (cnt <= 8) run(std::integral_constant<int, 8>());
      else run(std::integral_constant<int, 16>());
      __syncwarp();  // the next entry may add to the same token from other lanes
      q += g1 - g0;
    }
  }
  cl.sync();
  const int row0 = blockIdx.x / cs * 16 * MOE_W;
  for (int i = rank * 32 * MOE_W + threadIdx.x; i < a.N * 16 * MOE_W; i += cs * 32 * MOE_W) {
    float v = 0.0f;
    for (int c = 0; c < cs; ++c) v += cl.map_shared_rank(ypart, c)[i];
    const int n = i / (16 * MOE_W), row = row0 + i % (16 * MOE_W);
    if (row < a.K) {
      const int64_t o = (int64_t)n * a.ldy + row;
      if (ydt == 0) static_cast<float*>(a.y)[o] = v;
      else if (ydt == 1) static_cast<__nv_bfloat16*>(a.y)[o] = __float2bfloat16(v);
      else static_cast<__half*>(a.y)[o] = __float2half(v);
    }
  }
  cl.sync();  // no CTA leaves while another reads its part
}

// ------------------------------------------------------------ expert tiles
// One warp per group: 16 rows (of one matrix, or 8 of each of two) x 128
// columns of one expert; blocks past the last column get zeros.
template <int FMT>
__global__ void __launch_bounds__(256) k_moe_tile(const uint8_t* q, const unsigned short* d,
                                                  const uint8_t* q2, const unsigned short* d2,
                                                  int64_t ngroups, int rows, int cols,
                                                  uint8_t* out) {
  constexpr int GB = grp_bytes<FMT>();
  const int64_t wid = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (wid >= ngroups) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int kg = groups_of(cols), nb = cols / QK;
  const int64_t qrow = FMT == 8 ? cols : cols / 2;
  const int tiles = q2 ? rows / 8 : rows / 16;
  const int grp = (int)(wid % kg);
  const int64_t tl = wid / kg, e = tl / tiles, rt = tl % tiles;
  // rows g and g + 8 of the tile
  const int64_t r0 = e * rows + (q2 ? rt * 8 + g : rt * 16 + g);
  const int64_t r1 = q2 ? r0 : r0 + 8;
  const uint8_t* qa = q + r0 * qrow;
  const uint8_t* qb = (q2 ? q2 : q) + r1 * qrow;
  const unsigned short* da = d + r0 * nb;
  const unsigned short* db = (q2 ? d2 : d) + r1 * nb;
  uint8_t* o = out + wid * GB;
  uint32_t w[4][4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int blk = grp * 4 + b;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[b][j] = 0u;
    if (blk < nb) {
      if (FMT == 8) {
        w[b][0] = *reinterpret_cast<const uint32_t*>(qa + blk * 32 + t * 4);
        w[b][1] = *reinterpret_cast<const uint32_t*>(qb + blk * 32 + t * 4);
        w[b][2] = *reinterpret_cast<const uint32_t*>(qa + blk * 32 + 16 + t * 4);
        w[b][3] = *reinterpret_cast<const uint32_t*>(qb + blk * 32 + 16 + t * 4);
      } else {
        w[b][0] = *reinterpret_cast<const uint32_t*>(qa + blk * 16 + t * 4) ^ 0x88888888u;
        w[b][1] = *reinterpret_cast<const uint32_t*>(qb + blk * 16 + t * 4) ^ 0x88888888u;
      }
    }
  }
  if (FMT == 8) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<uint4*>(o + b * 512 + lane * 16) = make_uint4(w[b][0], w[b][1], w[b][2], w[b][3]);
  } else {
#pragma unroll
    for (int p = 0; p < 2; ++p)
      *reinterpret_cast<uint4*>(o + p * 512 + lane * 16) =
          make_uint4(w[2 * p][0], w[2 * p][1], w[2 * p + 1][0], w[2 * p + 1][1]);
  }
  // scales: [row g][block][row, row + 8]; lane (g, t) writes block t
  const int blk = grp * 4 + t;
  const uint32_t s = blk < nb ? (uint32_t)da[blk] | (uint32_t)db[blk] << 16 : 0u;
  *reinterpret_cast<uint32_t*>(o + grp_q<FMT>() + g * 16 + t * 4) = s;
}

struct WsMap {
  size_t ids, weights, xdig, xs, hdig, hs, bytes;
};
WsMap ws_map(int64_t N, int slots, int64_t K, int64_t F) {
  auto up = [](size_t v) { return (v + 127) / 128 * 128; };
  const size_t n = (size_t)std::min<int64_t>(N, MOE_NT), kg = groups_of(K), fg = groups_of(F);
  WsMap m;
  size_t o = 0;
  m.ids = o;
  o += up(n * slots * 4);
  m.weights = o;
  o += up(n * slots * 4);
  m.xdig = o;
  o += up(n * kg * MOE_DIG);
  m.xs = o;
  o += up(n * kg * 16);
  m.hdig = o;
  o += up(n * slots * fg * MOE_DIG);
  m.hs = o;
  o += up(n * slots * fg * 16);
  m.bytes = o;
  return m;
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

template <int TN>
size_t route_smem(int E) {
  const int epad = (E + RT_CL - 1) / RT_CL;
  return (size_t)TN * rt_chunk<TN>() * 8 + (size_t)RT_WARPS * epad * TN * 8 + (size_t)E * 12;
}

// Routing and / or the fixed-point form of x: one launch.
int launch_route(const MoeArgs& a, RouteArgs r, bool route, bool prep, const DeviceInfo& dev,
                 cudaStream_t st) {
  const int tn = a.N == 1 ? 1 : 8;
  r.clusters = route ? (a.N + tn - 1) / tn : 0;
  // one warp per token and group, at most two CTAs per SM, in whole clusters
  int pre = 0;
  if (prep) {
    const int64_t warps = (int64_t)a.N * groups_of(a.K);
    pre = (int)std::min<int64_t>((warps + RT_WARPS - 1) / RT_WARPS, 2 * dev.sms);
    pre = (pre + RT_CL - 1) / RT_CL * RT_CL;
  }
  const dim3 grid(RT_CL * r.clusters + pre);
  const void* f = tn == 1 ? (const void*)k_moe_route<1> : (const void*)k_moe_route<8>;
  if (int rc = allow_max_smem(f, dev)) return rc;
  const size_t smem = route ? (tn == 1 ? route_smem<1>(r.E) : route_smem<8>(r.E)) : 0;
  if (tn == 1) return launch("k_moe_route", k_moe_route<1>, grid, RT_THREADS, smem, RT_CL, st, a, r);
  return launch("k_moe_route", k_moe_route<8>, grid, RT_THREADS, smem, RT_CL, st, a, r);
}

template <int FMT>
int launch_up(const MoeArgs& a, const DeviceInfo& dev, cudaStream_t st) {
  if (int rc = allow_max_smem((const void*)k_moe_up<FMT>, dev)) return rc;
  const size_t smem = (size_t)MOE_W * ring_depth<FMT>() * grp_bytes<FMT>() +
                      table_bytes(a.E, a.N * a.slots, a.max_ent);
  int occ = 0;
  if (int rc = occupancy((const void*)k_moe_up<FMT>, dev, 32 * MOE_W, smem, &occ)) return rc;
  const int64_t units = (int64_t)a.max_ent * (a.F / 32);
  const dim3 grid((unsigned)std::min<int64_t>(units, (int64_t)dev.sms * occ));
  return launch("k_moe_up", k_moe_up<FMT>, grid, 32 * MOE_W, smem, 0, st, a);
}

template <int FMT>
int launch_down(const MoeArgs& a, int ydt, const DeviceInfo& dev, cudaStream_t st) {
  if (int rc = allow_max_smem((const void*)k_moe_down<FMT>, dev)) return rc;
  const size_t smem = (size_t)MOE_W * ring_depth<FMT>() * grp_bytes<FMT>() +
                      (size_t)a.N * 16 * MOE_W * 4 + table_bytes(a.E, a.N * a.slots, a.max_ent);
  const int chunks = (a.K / 16 + MOE_W - 1) / MOE_W;
  int cs = 1;  // CTAs that share 64 rows: as many as the device holds at once
  while (cs < 8 && chunks * cs * 2 <= dev.sms * 4) cs *= 2;
  return launch("k_moe_down", k_moe_down<FMT>, dim3(chunks * cs), 32 * MOE_W, smem, cs, st, a, ydt);
}

}  // namespace

size_t moe_tiles_bytes(int fmt, int64_t E, int64_t rows, int64_t cols) {
  const size_t gb = fmt == 8 ? grp_bytes<8>() : grp_bytes<4>();
  return (size_t)E * (rows / 16) * groups_of(cols) * gb;
}

int moe_tile(int fmt, const void* q, const void* d, const void* q2, const void* d2, int64_t E,
             int64_t rows, int64_t cols, void* out, cudaStream_t st) {
  const int64_t groups = E * (q2 ? rows / 8 : rows / 16) * groups_of(cols);
  const unsigned grid = (unsigned)((groups + 7) / 8);
  auto u8 = [](const void* p) { return static_cast<const uint8_t*>(p); };
  auto u16 = [](const void* p) { return static_cast<const unsigned short*>(p); };
  if (fmt == 8)
    k_moe_tile<8><<<grid, 256, 0, st>>>(u8(q), u16(d), u8(q2), u16(d2), groups, (int)rows,
                                        (int)cols, static_cast<uint8_t*>(out));
  else
    k_moe_tile<4><<<grid, 256, 0, st>>>(u8(q), u16(d), u8(q2), u16(d2), groups, (int)rows,
                                        (int)cols, static_cast<uint8_t*>(out));
  return check_launch("k_moe_tile");
}

size_t moe_workspace_bytes(int64_t N, int slots, int64_t K, int64_t F) {
  return ws_map(N, slots, K, F).bytes;
}

int moe_route(const MoeRoute& c, const void* x, int xdt, int64_t ldx, int64_t N, int64_t K,
              int* ids, float* weights, cudaStream_t st) {
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  // clusters of one launch are counted in 32 bits with room to spare
  constexpr int64_t kStep = (int64_t)1 << 20;
  for (int64_t n0 = 0; n0 < N; n0 += kStep) {
    MoeArgs a = {};
    const int64_t xb = xdt == 0 ? 4 : 2;
    a.x = static_cast<const uint8_t*>(x) + n0 * ldx * xb;
    a.ldx = ldx;
    a.xdt = xdt;
    a.N = (int)std::min(kStep, N - n0);
    RouteArgs r = {};
    r.w = c.w;
    r.wdt = c.wdt;
    r.ldw = c.ldw;
    r.bias = c.bias;
    r.E = c.E;
    r.K = (int)K;
    r.k = c.k;
    r.scoring = c.scoring;
    r.normalize = c.normalize;
    r.scale = c.scale;
    r.ids = ids + n0 * c.k;
    r.weights = weights + n0 * c.k;
    if (int rc = launch_route(a, r, true, false, dev, st)) return rc;
  }
  return OK;
}

int moe_experts(const MoeExperts& m, const MoeRoute* route, const void* x, int xdt, int64_t ldx,
                const int* ids, const float* weights, int slots, int64_t N, void* y, int64_t ldy,
                void* ws, cudaStream_t st) {
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  const WsMap wm = ws_map(N, slots, m.K, m.F);
  uint8_t* w = static_cast<uint8_t*>(ws);
  const int64_t xb = xdt == 0 ? 4 : 2;
  for (int64_t n0 = 0; n0 < N; n0 += MOE_NT) {
    MoeArgs a = {};
    a.x = static_cast<const uint8_t*>(x) + n0 * ldx * xb;
    a.ldx = ldx;
    a.xdt = xdt;
    a.N = (int)std::min<int64_t>(MOE_NT, N - n0);
    a.slots = slots;
    a.xdig = w + wm.xdig;
    a.xs = reinterpret_cast<float*>(w + wm.xs);
    a.hdig = w + wm.hdig;
    a.hs = reinterpret_cast<float*>(w + wm.hs);
    a.ids = route ? reinterpret_cast<int*>(w + wm.ids) : ids + n0 * slots;
    a.weights = route ? reinterpret_cast<float*>(w + wm.weights) : weights + n0 * slots;
    a.gate_up = static_cast<const uint8_t*>(m.gate_up);
    a.down = static_cast<const uint8_t*>(m.down);
    a.E = m.E;
    a.K = (int)m.K;
    a.F = (int)m.F;
    // every entry but an expert's last is full
    const int P = a.N * slots;
    a.max_ent = std::min(m.E, P) + P / MOE_ENT;
    a.y = static_cast<uint8_t*>(y) + n0 * ldy * xb;
    a.ldy = ldy;
    RouteArgs r = {};
    if (route) {
      r.w = route->w;
      r.wdt = route->wdt;
      r.ldw = route->ldw;
      r.bias = route->bias;
      r.E = route->E;
      r.K = (int)m.K;
      r.k = route->k;
      r.scoring = route->scoring;
      r.normalize = route->normalize;
      r.scale = route->scale;
      r.shared = slots - route->k;
      r.ids = reinterpret_cast<int*>(w + wm.ids);
      r.weights = reinterpret_cast<float*>(w + wm.weights);
    }
    if (int rc = launch_route(a, r, route != nullptr, true, dev, st)) return rc;
    if (int rc = m.fmt == 8 ? launch_up<8>(a, dev, st) : launch_up<4>(a, dev, st)) return rc;
    if (int rc = m.fmt_down == 8 ? launch_down<8>(a, xdt, dev, st) : launch_down<4>(a, xdt, dev, st))
      return rc;
  }
  return OK;
}

}  // namespace qg
