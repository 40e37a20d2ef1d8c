// Mixture-of-experts layer for a few tokens: router, SwiGLU experts in q8_0 /
// q4_0, and the weighted sum over each token's experts.
//
//   logits[n][e] = sum_k x[n][k] router[e][k]
//   ids[n][:], w[n][:] = the k best experts of token n and their weights
//   h[n][j] = w[n][j] silu(gate_e x_n) (up_e x_n),  e = ids[n][j]
//   y[n] = sum_j down_e h[n][j]
//
// Three launches, chained by programmatic dependent launch (no kernel waits on
// another's blocks, no counters, no atomics on global memory; each reads global
// memory only after its own dependency wait):
//
//  * k_moe_route: a cluster of CTAs per 1, 2 or 16 tokens; logits in 64-bit sums,
//    rounded to fp32 once (so the choice of experts does not depend on the
//    order of the sum), exchanged through distributed shared memory, then the
//    top k of each token by one warp.  Further CTAs of the same launch round x
//    to block fixed point (below).
//  * k_moe_up: work units of one expert x 32 h rows.  A warp's 16-row MMA tile is
//    8 gate rows and the same 8 up rows; the unit's 32 h values of a token are
//    one block of the down projection and are rounded to fixed point right
//    there.
//  * k_moe_down: a CTA owns 64 rows of y; a cluster of CTAs splits the chosen
//    experts' columns and adds its parts through distributed shared memory in
//    rank order (deterministic).
//
// Both stream their weights the same way: one CTA per SM, a producer warp that
// fills a ring of 9 stages with bulk copies (a stage is a slab: 4 row tiles x 2
// or 4 groups of 128 columns, 17 or 18 KB in one contiguous piece), and 12
// compute warps, one per row tile and one of three splits: split s takes every
// third slab.  Every wait is bounded.  What bounds them (one B200; the copy rate
// is 6.54 TB/s): with few tokens per expert q8_0 the weights' stream (16 tokens,
// 64 + 2 experts of 4096x1408: 971 MB in 192 us, 0.77 of the copy rate); q4_0 with
// several tokens the latency of a slab's digits and shared-memory loads, with four
// warps a scheduler (64 tokens, 128 experts of 2048x768, 335 MB in 159 us, 0.32:
// gate / up at 2.3 of 4 instructions per cycle, stalled on loads for 2.1 cycles per
// instruction and on fixed latencies for 1.5, down at 1.8); a single token the
// launches' latencies (128 experts of 2048x768 in q4_0, 8 chosen, 22 MB: 21.7 us).
// Tried and slower, when 16-bit types had two digits: 16 compute warps of 96
// registers (64 tokens 105 -> 156 us, spills), four MMAs of tokens per entry
// (spills), units of their own for the splits (64 tokens 105 -> 103 us, one token
// 20 -> 22), private rings of 16 warps without a producer (149 us).
//
// The arithmetic is the library's exact-integer scheme.  A block of 32
// activations is rounded to integers X = rint(x FX / max |x|) and split into
// signed byte digits X = p0 + 2^8 p1 + 2^16 p2; the integer dots of the
// block's quants with the digits are exact (mma.sync.m16n8k32.s8,
// |S| <= 32 * 128 * 128 = 2^19), and each block is scaled once:
// acc += (S0 + 2^8 S1 + 2^16 S2) (d max / FX).
//
// FX = 0x7F7F7F for every type of x and for h: a step of max |x| 2^-23 (the
// GEMVs' powers of two leave 2^-22 to 2^-21, and here two products follow one
// another: measured 7.5e-7 -> 2.9e-7 relative error of y).  bf16 and fp16
// activations do not get by with two digits, though two carry all their bits:
// the step is the block's, 2^-15 of its largest value then, and an outlier
// 1000 times its neighbours leaves them 1.5 % off, in full where a row's weight
// on the outlier is 0.  (The third digit costs bf16 nothing at one token, 6 % at
// 16 tokens over 64 experts in q8_0, 184 -> 195 us, and most where the
// instructions count: 64 tokens, 128 experts in q4_0, 115 -> 158 us.)
//
// The 8 columns of an MMA are the digits of 2 tokens, so one MMA per block
// serves up to 2, and a lane's pair of accumulators is one token's two low
// digits, joined as integers (|S0 + 2^8 S1| < 2^28) and converted once, or its
// high digit.
// A block that holds a NaN or an infinity gets a NaN scale: y is NaN there.
//
// Weights are "expert tiles", laid out once: per expert, chunks of 64 rows (four
// 16-row tiles; rows past the last are zero); a chunk's groups of 128 columns
// follow one another, each the four tiles' pieces; a tile's piece is its four
// blocks' quants in MMA fragment order (one 16-byte shared-memory load per lane
// is a q8_0 A fragment, or two of q4_0) and then the scales [8 rows][4 blocks]
// [row, row + 8].  q4_0 nibbles are stored with bit 3 flipped: n ^ 8 shifted
// into the high half of a byte is 16 (n - 8) as a signed byte, one or two
// instructions; the 1/16 is folded into the result's factor (exact).
#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "qgemv_common.cuh"
#include "qgemv_internal.h"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace qg {

__device__ int g_moe_error = 0;
__device__ long long g_moe_spin_limit = kDefaultSpinLimit;

namespace {

constexpr int MOE_NT = kMoeTokens;  // tokens per pass
constexpr int MOE_RT = 4;                  // row tiles (of 16) of a slab, one per compute warp
constexpr int MOE_KS = 3;                  // compute warps per row tile
constexpr int MOE_CW = MOE_RT * MOE_KS;    // compute warps; then the producer
constexpr int MOE_EW = 3;                  // gate / up: warps that finish units
constexpr int UP_THREADS = 32 * (MOE_CW + 1 + MOE_EW);
constexpr int DN_THREADS = 32 * (MOE_CW + 1);
constexpr int MOE_DOWN_CL = 8;             // down: CTAs of a cluster, at most
constexpr int MOE_GCOLS = 128;      // columns of a group (4 blocks)
// digit bytes of a group: [digits][4 lanes][32]
constexpr int MOE_DIG = 3;
constexpr int DIG_BYTES = MOE_DIG * 128;
// tokens that share one MMA, and of one entry (one or two MMAs) at most: four
// MMAs an entry do not fit the registers (they spilled 1 KB and cost all
// calls 1.5x); an expert with more tokens streams its weights again, from L2
constexpr int TOK_MMA = 2, MOE_ENT = 2 * TOK_MMA;

// bytes of a group (16 rows x 128 columns): quants, then 64 fp16 scales
template <int FMT> __host__ __device__ constexpr int grp_q() { return FMT == 8 ? 2048 : 1024; }
template <int FMT> __host__ __device__ constexpr int grp_bytes() { return grp_q<FMT>() + 128; }
// A slab: 4 row tiles x SG groups; 9 stages are 153 or 162 KB.  The number of
// stages is a multiple of the splits, so that a stage always belongs to the
// same split: a warp knows a barrier's phase from its own slabs only.
constexpr int MOE_S = 9;
static_assert(MOE_S % MOE_KS == 0, "a stage serves one split");
template <int FMT> __host__ __device__ constexpr int slab_groups() { return FMT == 8 ? 2 : 4; }
template <int FMT> __host__ __device__ constexpr int slab_bytes() { return MOE_RT * slab_groups<FMT>() * grp_bytes<FMT>(); }
template <int FMT> __host__ __device__ constexpr int ring_bytes() { return MOE_S * slab_bytes<FMT>(); }

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
constexpr int FX_MAX = 0x7F7F7F;  // every signed byte digit at most 127
__device__ __forceinline__ BlockScale block_scale(uint32_t amax) {
  constexpr float FX = (float)FX_MAX;
  BlockScale b{1.0f, 0.0f, 0.0f};
  const float m = __uint_as_float(amax);
  if (amax >= 0x7F800000u) {
    b.scale = __int_as_float(0x7FC00000);
  } else if (amax != 0u) {
    const bool tiny = m < 5.421010862427522e-20f;  // 2^-64
    b.up = tiny ? 18446744073709551616.0f : 1.0f;
    b.s = FX / (m * b.up);
    b.scale = m * b.up / FX * (tiny ? 5.421010862427522e-20f : 1.0f);
  }
  return b;
}
// X + 0x808080 of one value: byte p, with its top bit flipped, is
// digit p.  The clamp holds |X| <= FX also where the product rounds up, so the
// biased value keeps to its digits.  A value of a non-finite block gives 0.
__device__ __forceinline__ uint32_t fixed_biased(float v, const BlockScale& b) {
  const int X = b.s == 0.0f ? 0 : __float2int_rn(v * b.up * b.s);
  return (uint32_t)(min(max(X, -FX_MAX), FX_MAX) + 0x808080);
}

struct MoeArgs {
  // activations and their fixed-point form
  const void* x;
  int64_t ldx;
  int xdt;
  uint8_t* xdig;   // [N][K groups][digit bytes]
  float* xs;       // [N][K groups * 4]
  uint8_t* hdig;   // [N * slots][F groups][digit bytes]
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
  int clusters;    // CTAs [0, cluster size * clusters) route; the others prepare x
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
    uint8_t* dst = a.xdig + (int64_t)i * DIG_BYTES + t * 32 + blk * 8 + half * 4;
#pragma unroll
    for (int p = 0; p < MOE_DIG; ++p) {
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
// CTAs of a routing cluster that takes TN tokens (16 is the opt-in size; a
// single token's logits are all latency, so they are spread widest)
template <int TN> __host__ __device__ constexpr int rt_cl() { return TN == 1 ? 16 : 8; }
constexpr int RT_TE = 4;    // experts of a warp's tile
// x columns staged at a time, as doubles (32 KB)
template <int TN> __host__ __device__ constexpr int rt_chunk() { return TN == 1 ? 4096 : 2048; }

// Ordering keys of a score: larger key = larger score, +0 == -0, NaN lowest (1;
// 0 marks a taken expert).
__device__ __forceinline__ unsigned long long rank_key(double v) {
  if (v != v) return 1ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t rank_key(float v) {
  if (v != v) return 1u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
// The largest key of the warp's lanes.
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = (uint32_t)(k >> 32), mh = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t ml = __reduce_max_sync(0xffffffffu, hi == mh ? (uint32_t)k : 0u);
  return (unsigned long long)mh << 32 | ml;
}
// k rounds over E keys in shared memory; lane j returns the j-th choice.  Lane
// l's experts are l, l + 32, ...; equal keys go to the lowest expert.
template <typename Key>
__device__ __forceinline__ int pick(Key* key, int E, int k, int lane) {
  int mine = 0;
  for (int j = 0; j < k; ++j) {
    Key best = 0;
    int at = lane;
#pragma unroll 4
    for (int e = lane; e < E; e += 32)
      if (key[e] > best) {
        best = key[e];
        at = e;
      }
    const Key top = warp_max(best);
    const int win = (int)__reduce_min_sync(0xffffffffu, best == top ? (uint32_t)at : 0xFFFFFFFFu);
    if (lane == j) mine = win;
    if (win == at) key[win] = 0;
    __syncwarp();
  }
  return mine;
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

// The top k of one token by one warp: `logit` holds E values in shared memory,
// `key` room for as many 64-bit keys.  (A token's choice is latency and little
// else, run once per launch from a cold instruction cache: short loops.)
__device__ void route_token(const RouteArgs& r, const float* logit, unsigned long long* key, int n, int lane) {
  const int E = r.E, slots = r.k + r.shared;
  uint32_t* key32 = reinterpret_cast<uint32_t*>(key);
  float mx = -INFINITY;
  bool nan = false;
  for (int e = lane; e < E; e += 32) {
    const float l = logit[e];
    mx = fmaxf(mx, l);
    nan |= l != l;
    key32[e] = rank_key(l);
  }
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  nan = __any_sync(0xffffffffu, nan);
  __syncwarp();
  int mine;
  if (!r.bias) {
    // softmax and sigmoid are increasing: the logits rank the experts
    mine = pick(key32, E, r.k, lane);
  } else {
    // with a bias the scores are formed in 64 bits, so that rounding does not
    // decide between near scores
    double all = 0.0;
    if (r.scoring == 0) {
      for (int e = lane; e < E; e += 32) all += exp((double)logit[e] - (double)mx);
      for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    for (int e = lane; e < E; e += 32) {
      const double l = (double)logit[e];
      key[e] = rank_key((r.scoring == 0 ? exp(l - (double)mx) / all : 1.0 / (1.0 + exp(-l))) + (double)r.bias[e]);
    }
    __syncwarp();
    mine = pick(key, E, r.k, lane);
  }
  float s = 0.0f, top = mx;
  if (r.bias && r.normalize && r.scoring == 0) {
    // the bias may have chosen experts far below the best one: their weights
    // are relative to each other, so to the largest of them
    float c = lane < r.k ? logit[mine] : -INFINITY;
    for (int o = 16; o; o >>= 1) c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, o));
    if (c != -INFINITY) top = c;
  }
  if (lane < r.k) {
    const float l = logit[mine];
    s = r.scoring == 0 ? expf(l - top) : 1.0f / (1.0f + expf(-l));
  }
  const float sum = warp_sum(s);
  // scores are fp32 numbers: where every chosen one is 0 the weights are, not NaN
  float den = r.normalize && sum > 0.0f ? sum : 1.0f;
  if (!r.normalize && r.scoring == 0) {
    float all = 0.0f;
    for (int e = lane; e < E; e += 32) all += expf(logit[e] - mx);
    den = warp_sum(all);
  }
  if (lane < r.k) {
    r.ids[(int64_t)n * slots + lane] = mine;
    r.weights[(int64_t)n * slots + lane] = nan || sum != sum ? __int_as_float(0x7FC00000) : s / den * r.scale;
  } else if (lane < slots) {
    r.ids[(int64_t)n * slots + lane] = E + lane - r.k;
    r.weights[(int64_t)n * slots + lane] = 1.0f;
  }
}

// CTAs [0, CL * clusters): cluster c routes tokens [TN c, TN c + TN), CTA rank
// r computing the logits of experts [E r / CL, E (r + 1) / CL) and choosing for
// token TN c + r.  A warp takes tiles of 4 experts x TN tokens; with fewer
// tiles than warps the columns are split over them too.  The sums are in
// fp64 (measured here: 64 FMA per clock and SM, the conversions from fp32 a
// quarter of that, which is why x is converted once per CTA).
template <int TN>
__global__ void __launch_bounds__(RT_THREADS, 2) k_moe_route(MoeArgs a, RouteArgs r) {
  extern __shared__ __align__(16) uint8_t rt_smem[];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int RT_CL = rt_cl<TN>();
  if ((int)blockIdx.x >= RT_CL * r.clusters) {
    pdl_wait();
    const int w = (blockIdx.x - RT_CL * r.clusters) * RT_WARPS + warp;
    const int nw = (gridDim.x - RT_CL * r.clusters) * RT_WARPS;
    prepare_x(a, w, nw, lane);
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
  auto started = cl.barrier_arrive();  // this CTA runs: its shared memory may be written to
  const int tiles = (ne + RT_TE - 1) / RT_TE;
  int ks = 1;  // warps that share a tile's columns
  while (ks < RT_WARPS && ks * 2 * tiles <= RT_WARPS) ks *= 2;
  const int sl = warp % ks;
  pdl_wait();
  const bool vec = r.ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(r.w) & 15) == 0;
  const bool xvec = a.ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  for (int t0 = 0; t0 < tiles; t0 += RT_WARPS / ks) {
    const int tl = t0 + warp / ks, eb = e0 + tl * RT_TE;
    double acc[RT_TE * TN] = {};
    auto load = [&](float (&w)[RT_TE][4], int c) {
#pragma unroll
      for (int i = 0; i < RT_TE; ++i)
        load4(w[i], r.w, r.wdt, (int64_t)min(eb + i, e1 - 1) * r.ldw + c + 4 * lane, K - c - 4 * lane, vec);
    };
    auto step = [&](const float (&w)[RT_TE][4], int cb) {
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
    };
    // the first steps' weights are on their way while x is staged
    constexpr int PRE = TN == 1 ? 4 : 2;
    float pre[PRE][RT_TE][4];
    if (tl < tiles)
#pragma unroll
      for (int j = 0; j < PRE; ++j)
        if ((sl + j * ks) * 128 < min(CH, K)) load(pre[j], (sl + j * ks) * 128);
    for (int c0 = 0; c0 < K; c0 += CH) {
      const int cn = min(CH, K - c0);
      __syncthreads();
      // column 128 i + 4 l + j sits at 128 i + 64 (j / 2) + 2 l + j % 2: a lane
      // reads its four columns with two conflict-free 16-byte loads
      const int cr = (cn + 127) & ~127;
      for (int n = 0; n < TN; ++n)
#pragma unroll 4
        for (int c = threadIdx.x * 4; c < cr; c += RT_THREADS * 4) {
          float v[4];
          load4(v, a.x, a.xdt, (int64_t)(n0 + min(n, nn - 1)) * a.ldx + c0 + c, n < nn ? cn - c : 0, xvec);
          double* d = xd + n * CH + (c & ~127) + ((c >> 2) & 31) * 2;
          *reinterpret_cast<double2*>(d) = make_double2((double)v[0], (double)v[1]);
          *reinterpret_cast<double2*>(d + 64) = make_double2((double)v[2], (double)v[3]);
        }
      __syncthreads();
      if (tl < tiles) {
        int j = 0;
        if (c0 == 0) {
#pragma unroll
          for (; j < PRE; ++j)
            if ((sl + j * ks) * 128 < cn) step(pre[j], (sl + j * ks) * 128);
        }
#pragma unroll 2
        for (int cb = (sl + j * ks) * 128; cb < cn; cb += ks * 128) {
          float w[RT_TE][4];
          load(w, c0 + cb);
          step(w, cb);
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
  __syncthreads();  // every partial sum is there
  cl.barrier_wait(std::move(started));
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

// Many tokens: clusters of 8 CTAs take 16 tokens; a warp 16 experts x 16 tokens
// of a slice of the columns, on the fp64 matrix instruction m8n8k4 (the same 64
// multiply-adds per clock and SM as DFMA, but two operand registers for 256 of
// them): lane (r, t) reads four consecutive columns 4t ... of rows r and r + 8 of
// both matrices straight into fragments, so nothing is staged.
constexpr int RM_TN = 16, RM_CL = 8, RM_TE = 16;
// Four columns of a row as they were read: a row that can be read in vectors
// keeps its type until it is used, so that the loads of the next steps are in
// flight meanwhile (converted at once, each step waited for its loads: 512 tokens,
// 256 experts of 4096 columns took 120 us, now 60).
struct Raw4 {
  uint32_t v[4];
  __device__ __forceinline__ void load(const void* p, int dt, int64_t i, int n, bool vec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0u;
    if (n <= 0) return;
    if (!vec) {
      for (int j = 0; j < 4; ++j)
        if (j < n) v[j] = __float_as_uint(load_as_f32(p, dt, i + j));
    } else if (dt == 0) {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
      v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
      v[0] = u.x, v[1] = u.y;
    }
  }
  // fmt: the row's type, or 0 where load() converted already
  __device__ __forceinline__ void get(float (&f)[4], int fmt) const {
    if (fmt == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t h = j & 1 ? v[j >> 1] >> 16 : v[j >> 1] & 0xFFFFu;
        f[j] = fmt == 1 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
      }
    }
  }
};
__device__ __forceinline__ void dmma(double (&c)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
      : "+d"(c[0]), "+d"(c[1])
      : "d"(a), "d"(b));
}
__host__ __device__ constexpr int rm_slices(int ne) {  // warps that share a tile's columns
  int ks = 1;
  while (ks < RT_WARPS && ks * 2 * ((ne + RM_TE - 1) / RM_TE) <= RT_WARPS) ks *= 2;
  return ks;
}
__global__ void __launch_bounds__(RT_THREADS, 2) k_moe_route_many(MoeArgs a, RouteArgs r) {
  extern __shared__ __align__(16) uint8_t rt_smem[];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((int)blockIdx.x >= RM_CL * r.clusters) {
    pdl_wait();
    const int w = (blockIdx.x - RM_CL * r.clusters) * RT_WARPS + warp;
    const int nw = (gridDim.x - RM_CL * r.clusters) * RT_WARPS;
    prepare_x(a, w, nw, lane);
    return;
  }
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), E = r.E, K = r.K;
  const int n0 = (blockIdx.x / RM_CL) * RM_TN, nn = min(RM_TN, a.N - n0);
  const int e0 = (int)((int64_t)E * rank / RM_CL), e1 = (int)((int64_t)E * (rank + 1) / RM_CL);
  const int ne = e1 - e0, epad = (E + RM_CL - 1) / RM_CL;
  // shared memory: keys of two tokens [2][E], partial sums [slices][epad][16],
  // the logits of this CTA's tokens (rank and rank + 8) [2][E]
  const int kmax = rm_slices(epad);  // the same layout in every CTA of the cluster
  unsigned long long* key = reinterpret_cast<unsigned long long*>(rt_smem);
  double* part = reinterpret_cast<double*>(key + 2 * E);
  float* logit = reinterpret_cast<float*>(part + kmax * epad * RM_TN);
  auto started = cl.barrier_arrive();  // this CTA runs: its shared memory may be written to
  const int tiles = (ne + RM_TE - 1) / RM_TE, ks = kmax, sl = warp % ks;
  const int row = lane >> 2, t = lane & 3;
  const bool vec = K % 4 == 0 && r.ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(r.w) & 15) == 0;
  const bool xvec = K % 4 == 0 && a.ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  const int wfmt = vec ? r.wdt : 0, xfmt = xvec ? a.xdt : 0;
  pdl_wait();
  for (int tl = warp / ks; tl < tiles; tl += RT_WARPS / ks) {
    const int eb = e0 + tl * RM_TE;
    double acc[2][2][2] = {};
    const int64_t w0 = (int64_t)min(eb + row, e1 - 1) * r.ldw, w1 = (int64_t)min(eb + 8 + row, e1 - 1) * r.ldw;
    const int64_t x0 = (int64_t)(n0 + min(row, nn - 1)) * a.ldx, x1 = (int64_t)(n0 + min(8 + row, nn - 1)) * a.ldx;
    struct Step {
      Raw4 w[2], x[2];
    } ring[3];
    auto load = [&](Step& s, int cb) {
      const int c = cb + 4 * t, n = K - c;
      s.w[0].load(r.w, r.wdt, w0 + c, n, vec);
      s.w[1].load(r.w, r.wdt, w1 + c, n, vec);
      s.x[0].load(a.x, a.xdt, x0 + c, n, xvec);
      s.x[1].load(a.x, a.xdt, x1 + c, n, xvec);
    };
    const int step = ks * 16;
    load(ring[0], sl * 16);
    load(ring[1], sl * 16 + step);
    for (int cb = sl * 16; cb < K; cb += 3 * step) {  // every lane takes part to the end
#pragma unroll
      for (int u = 0; u < 3; ++u) {
        if (cb + u * step >= K) break;
        load(ring[(u + 2) % 3], cb + (u + 2) * step);
        float fw[2][4], fx[2][4];
        ring[u].w[0].get(fw[0], wfmt);
        ring[u].w[1].get(fw[1], wfmt);
        ring[u].x[0].get(fx[0], xfmt);
        ring[u].x[1].get(fx[1], xfmt);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int q = 0; q < 2; ++q) dmma(acc[p][q], (double)fw[p][i], (double)fx[q][i]);
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int e = eb + 8 * p + row - e0, n = 8 * q + 2 * t + i;
          if (e < ne) part[(sl * epad + e) * RM_TN + n] = acc[p][q][i];
        }
  }
  __syncthreads();  // every partial sum is there
  cl.barrier_wait(std::move(started));
  for (int i = threadIdx.x; i < ne * nn; i += RT_THREADS) {
    const int e = i / nn, n = i % nn;
    double v = 0.0;
    for (int s = 0; s < ks; ++s) v += part[(s * epad + e) * RM_TN + n];
    cl.map_shared_rank(logit, n % RM_CL)[(n / RM_CL) * E + e0 + e] = (float)v;
  }
  cl.sync();
  if (warp < RM_TN / RM_CL && rank + RM_CL * warp < nn)
    route_token(r, logit + warp * E, key + warp * E, n0 + rank + RM_CL * warp, lane);
}

// --------------------------------------------------- entries of the experts
// The chosen experts in ascending order (one token's: in its order), each with up to MOE_ENT of its tokens
// (an expert with more has several entries), built by every CTA for itself from
// the choices.  A choice outside [0, E) selects nothing; an expert that one
// token names twice counts once, with the sum of the weights.  An expert's
// tokens are kept as a 64-bit mask and taken in ascending order: every CTA
// builds the same entries, since the CTAs share them out.
struct Table {
  uint32_t* mask;   // [E][2] tokens of the expert
  int* first;       // [E]
  // [max_ent] expert | first << 10 | count << 22 | its place among the
  // expert's entries << 26 (64 tokens in entries of 4: 15 at most)
  uint32_t* ent;
  uint32_t* tmp;    // [P]
  uint32_t* sorted; // [P] choice | token << 16, by expert
  float* w;         // [P]
  int nent;
  // entries of entry e's expert
  __device__ __forceinline__ int run(int e) const {
    const uint32_t x = ent[e] & 1023u;
    const int c = __popc(mask[2 * x]) + __popc(mask[2 * x + 1]);
    return (c + MOE_ENT - 1) / MOE_ENT;
  }
};
__host__ __device__ __forceinline__ size_t table_bytes(int E, int P, int max_ent) {
  return (size_t)(3 * E + max_ent + 3 * P) * 4;
}

// No expert has tokens yet: before build_table, and before the choices are known.
__device__ __forceinline__ void clear_table(uint8_t* mem, const MoeArgs& a) {
  for (int i = threadIdx.x; i < 2 * a.E; i += blockDim.x) reinterpret_cast<uint32_t*>(mem)[i] = 0u;
  __syncthreads();
}
__device__ Table build_table(uint8_t* mem, const MoeArgs& a) {
  __shared__ uint32_t wsum[32];
  const int P = a.N * a.slots, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Table t;
  t.mask = reinterpret_cast<uint32_t*>(mem);
  t.first = reinterpret_cast<int*>(t.mask + 2 * a.E);
  t.ent = reinterpret_cast<uint32_t*>(t.first + a.E);
  t.tmp = t.ent + a.max_ent;
  t.sorted = t.tmp + P;
  t.w = reinterpret_cast<float*>(t.sorted + P);
  if (a.N == 1) {  // a lane per choice: an entry for each distinct expert, in their order
    if (warp == 0) {
      const uint32_t id = lane < P ? (uint32_t)a.ids[lane] : 0xFFFFFFFFu;
      const float w = lane < P ? a.weights[lane] : 0.0f;
      const uint32_t same = __match_any_sync(0xffffffffu, id);
      const bool keep = id < (uint32_t)a.E && lane == __ffs(same) - 1;
      const uint32_t kept = __ballot_sync(0xffffffffu, keep);
      float sum = 0.0f;
      for (int i = 0; i < P; ++i) {
        const float v = __shfl_sync(0xffffffffu, w, i);
        if ((same >> i) & 1u) sum += v;
      }
      if (keep) {
        const int i = __popc(kept & ((1u << lane) - 1u));
        t.ent[i] = id | (uint32_t)i << 10 | 1u << 22;
        t.sorted[i] = (uint32_t)lane;
        t.w[lane] = sum;
        t.mask[2 * id] = 1u;  // run() counts its tokens
      }
      if (lane == 0) wsum[0] = (uint32_t)__popc(kept);
    }
    __syncthreads();
    t.nent = (int)wsum[0];
      return t;
  }
  for (int p = tid; p < P; p += blockDim.x) {
    const uint32_t id = (uint32_t)a.ids[p];
    const int n = p / a.slots;
    t.tmp[p] = id;
    t.w[p] = a.weights[p];
    if (id < (uint32_t)a.E) atomicOr(&t.mask[2 * id + (n >> 5)], 1u << (n & 31));
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
  for (int i = 0; i < (int)blockDim.x / 32; ++i) {
    if (i < warp) before += wsum[i];
    total += wsum[i];
  }
  uint32_t c0 = before & 0xFFFFu, n0 = before >> 16;
  for (int i = b; i < e; ++i) {
    const uint32_t c = count(i);
    for (uint32_t j = 0; j < c; j += MOE_ENT)
      t.ent[n0++] = (uint32_t)i | (c0 + j) << 10 | min((uint32_t)MOE_ENT, c - j) << 22 | j / MOE_ENT << 26;
    t.first[i] = (int)c0;
    c0 += c;
  }
  __syncthreads();
  for (int p = tid; p < P; p += blockDim.x) {
    const uint32_t id = t.tmp[p];
    const int n = p / a.slots;
    bool keep = id < (uint32_t)a.E;  // the token's first choice of this expert
    for (int q = n * a.slots; q < p; ++q) keep &= t.tmp[q] != id;
    if (keep) {
      // its duplicates' weights are only read, their own entries not written
      float w = t.w[p];
      for (int q = p + 1; q < (n + 1) * a.slots; ++q)
        if (t.tmp[q] == id) w += t.w[q];
      t.w[p] = w;
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
__device__ __forceinline__ long long moe_spin_limit() {
  return *(volatile long long*)&g_moe_spin_limit;
}
// Bounded wait; gives up at once when another thread raised the abort flag.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const long long t0 = clock64(), lim = moe_spin_limit();
  while (!mbar_try(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > lim) {
      atomicExch(&g_moe_error, (int)ERR_TIMEOUT);
      __threadfence();
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_try(bar, parity) || wait_slow(bar, parity, abort_flag);
}
// The same by a whole warp, which goes on or gives up as one: a lane may see
// the barrier, another the abort flag, and what follows (warp-wide reductions,
// shuffles and MMAs, the cluster's barrier) wants every lane.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// Wait for a copy in flight before the CTA ends: ignores the abort flag,
// bounded by at least the default limit.
__device__ __noinline__ void drain(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64(), lim = max(moe_spin_limit(), kDefaultSpinLimit);
  while (!mbar_try(bar, parity) && clock64() - t0 < lim) {
  }
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
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0), "r"(0), "r"(0),
        "r"(0));
}

// The stages' barriers of a CTA, and the parts of a unit (gate and up).
struct Pipe {
  unsigned long long full[MOE_S], empty[MOE_S], pfull[2], pempty[2];
  int abort_flag;
  __device__ __forceinline__ void init() {
    for (int s = 0; s < MOE_S; ++s) {
      mbar_init(saddr(&full[s]), 1);
      mbar_init(saddr(&empty[s]), MOE_RT);  // the row tiles' warps of the slab's split
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(saddr(&pfull[b]), MOE_CW);
      mbar_init(saddr(&pempty[b]), MOE_EW);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
};

// A compute warp's place in the ring: stages kq, kq + 3, ... in turn.
struct Turn {
  int s;
  uint32_t phase = 0u;
  __device__ __forceinline__ void next() {
    s += MOE_KS;
    if (s >= MOE_S) {
      s -= MOE_S;
      phase ^= 1u;
    }
  }
};

// The producer thread's side: slab after slab into stages 0, 1, ...
template <int FMT>
struct Feed {
  Pipe& p;
  uint32_t ring;
  int i = 0;  // slabs so far
  // m groups at src; false once the launch gave up
  __device__ __forceinline__ bool put(const uint8_t* src, int m) {
    const int s = i % MOE_S;
    if (i >= MOE_S && !mbar_wait(saddr(&p.empty[s]), (uint32_t)(i / MOE_S - 1) & 1u, &p.abort_flag)) return false;
    const uint32_t bytes = (uint32_t)(m * MOE_RT * grp_bytes<FMT>());
    mbar_expect_tx(saddr(&p.full[s]), bytes);
    bulk_g2s(ring + s * slab_bytes<FMT>(), src, bytes, saddr(&p.full[s]));
    ++i;
    return true;
  }
  // no copy outlives the CTA, whatever the other warps gave up on
  __device__ __forceinline__ void finish() {
    for (int k = max(0, i - MOE_S); k < i; ++k) drain(saddr(&p.full[k % MOE_S]), (uint32_t)(k / MOE_S) & 1u);
  }
};

// A fragments (block i of the pair in a[i]) and scales (rows g and g + 8) of
// blocks 2 p and 2 p + 1 of the group at `st`.
template <int FMT>
struct Quants {
  uint32_t a[2][4];
  float2 d[2];
  __device__ __forceinline__ void load(uint32_t st, int p, int lane) {
    uint2 dv;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                 : "=r"(dv.x), "=r"(dv.y)
                 : "r"(st + grp_q<FMT>() + (lane >> 2) * 16 + p * 8)
                 : "memory");
    d[0] = __half22float2(*reinterpret_cast<const __half2*>(&dv.x));
    d[1] = __half22float2(*reinterpret_cast<const __half2*>(&dv.y));
    if (FMT == 8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = lds128(st + (2 * p + i) * 512 + lane * 16);
        a[i][0] = v.x;
        a[i][1] = v.y;
        a[i][2] = v.z;
        a[i][3] = v.w;
      }
    } else {
      // words: block 2 p (row g, row g + 8), block 2 p + 1 (row g, row g + 8)
      const uint4 v = lds128(st + p * 512 + lane * 16);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i >> 1][i & 1] = (w[i] << 4) & 0xF0F0F0F0u;    // columns 4t ...
        a[i >> 1][2 + (i & 1)] = w[i] & 0xF0F0F0F0u;     // columns 16 + 4t ...
      }
    }
  }
};

// The digits and block scales of one MMA's tokens for a group, as a lane
// holds them: its column lane / 4 is token (lane / 4) / (8 / tokens), the
// digit the rest; its accumulators belong to columns 2t and 2t + 1.
struct Digits {
  uint4 b[2];
  uint4 s;
};
// Where a lane finds the digits and scales of one MMA's tokens: group 0's.
struct Cols {
  const uint8_t* dig;
  const float* s;
  // row(i): the activation row of the i-th of `cnt` tokens; the columns of
  // absent tokens repeat the last one's
  template <typename Row>
  __device__ __forceinline__ void set(const uint8_t* digits, const float* scales, int groups, int cnt,
                                      int lane, Row row) {
    const int n = lane >> 2, t = lane & 3;
    // column 3 (and 7) is idle and reads digit 2 again; its accumulator is dropped
    const int tok = n >> 2, d = min(n & 3, 2);
    dig = digits + row(min(tok, cnt - 1)) * groups * DIG_BYTES + d * 128 + t * 32;
    s = scales + row(min(t >> 1, cnt - 1)) * groups * 4;
  }
  // group j from here
  __device__ __forceinline__ void load(Digits& f, int j) const {
    f.b[0] = ldg128(dig + j * DIG_BYTES);
    f.b[1] = ldg128(dig + j * DIG_BYTES + 16);
    f.s = ldg128(s + j * 4);
  }
  __device__ __forceinline__ Cols at(int grp) const {
    return Cols{dig + (int64_t)grp * DIG_BYTES, s + (int64_t)grp * 4};
  }
};

// acc[0], acc[1]: rows g and g + 8 of the lane's token (the even lane holds
// the two low digits' sum, the odd one the high digit's); blocks
// 2 p and 2 p + 1.  w: the second column's weight (256, or 0 in the odd lane).
template <int FMT>
__device__ __forceinline__ void product(float* acc, const Quants<FMT>& q, const Digits& f, int p, int w) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int c[4];
    mma_s8(c, q.a[i], i ? f.b[p].z : f.b[p].x, i ? f.b[p].w : f.b[p].y);
    const float sc = __uint_as_float(p == 0 ? (i ? f.s.y : f.s.x) : (i ? f.s.w : f.s.z));
    acc[0] = fmaf((float)(c[0] + c[1] * w), q.d[i].x * sc, acc[0]);
    acc[1] = fmaf((float)(c[2] + c[3] * w), q.d[i].y * sc, acc[1]);
  }
}

// What a compute warp holds: the digits of the slab at hand, read a slab ahead
// (they come from L2: a group ahead left the warps waiting), and its 16 rows'
// sums.  Four sets of digits fit the registers: two groups of one or two MMAs
// of tokens (q8_0), four groups of one MMA (q4_0); a q4_0 slab with two MMAs
// keeps two groups and reads on inside the slab.
template <int FMT>
struct Work {
  static constexpr int T = TOK_MMA, SG = slab_groups<FMT>();
  // the slab ahead: its tokens' digits (of its first group), groups and width
  struct Ahead {
    Cols c0, c1;
    int m = 0;  // 0: none
    bool two = false;
  };
  Cols e0, e1;  // the entry ahead, from its first group
  bool etwo;
  Digits f[4];
  float acc[4];
  // the next slabs' entry: its tokens; row(i) as in Cols
  template <typename Row>
  __device__ __forceinline__ void entry(const uint8_t* digits, const float* scales, int groups, int cnt,
                                        int lane, Row row) {
    etwo = cnt > T;
    e0.set(digits, scales, groups, cnt, lane, row);
    if (etwo) e1.set(digits, scales, groups, cnt - T, lane, [&](int i) { return row(T + i); });
  }
  __device__ __forceinline__ Ahead ahead(int grp, int m) const {
    Ahead a;
    a.c0 = e0.at(grp);
    a.c1 = e1.at(grp);
    a.m = m;
    a.two = etwo;
    return a;
  }
  __host__ __device__ static constexpr bool whole(bool two) { return SG == 2 || !two; }  // all of a slab's digits fit
  __host__ __device__ static constexpr int slot(bool two, int j, int c) {
    return SG == 2 ? j * 2 + c : two ? (j & 1) * 2 + c : j;
  }
  template <bool TWO>
  __device__ __forceinline__ void load(const Ahead& a, int j) {
    a.c0.load(f[slot(TWO, j, 0)], j);
    if (TWO) a.c1.load(f[slot(TWO, j, 1)], j);
  }
  // what a slab starts with
  __device__ __forceinline__ void begin(const Ahead& a) {
#pragma unroll
    for (int j = 0; j < SG; ++j) {
      if (j >= a.m) break;
      if (a.two) {
        if (whole(true) || j < 2) load<true>(a, j);
      } else {
        load<false>(a, j);
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
  }
  template <bool TWO>
  __device__ __forceinline__ void groups(uint32_t st, const Ahead& now, const Ahead& next, int lane) {
    const int w = lane & 1 ? 0 : 256;
    const int nm = whole(TWO) && next.two == TWO ? next.m : 0;
#pragma unroll
    for (int j = 0; j < SG; ++j) {
      if (j > 0 && j >= now.m) break;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        Quants<FMT> q;
        q.load(st + j * MOE_RT * grp_bytes<FMT>(), p, lane);
        product<FMT>(acc, q, f[slot(TWO, j, 0)], p, w);
        if (TWO) product<FMT>(acc + 2, q, f[slot(TWO, j, 1)], p, w);
      }
      if (whole(TWO)) {
        if (j < nm) load<TWO>(next, j);
      } else if (j + 2 < now.m) {
        load<TWO>(now, j + 2);
      }
    }
    // groups of a longer next slab that this one had none for, or all of them
    if (nm > 0) {
#pragma unroll
      for (int j = 1; j < SG; ++j)
        if (j >= now.m && j < nm) load<TWO>(next, j);
    } else {
      begin(next);
    }
  }
  // the slab `now`, whose digits are there or on their way; asks for `next`'s
  __device__ __forceinline__ void slab(uint32_t st, int rt, const Ahead& now, const Ahead& next, int lane) {
    st += rt * grp_bytes<FMT>();
    if (now.two) groups<true>(st, now, next, lane);
    else groups<false>(st, now, next, lane);
  }
  // put(token of the entry, row g's sum, row g + 8's sum) for every token that
  // this lane holds
  template <typename Put>
  __device__ __forceinline__ void each(int cnt, int lane, Put put) {
    constexpr float Q = FMT == 8 ? 1.0f : 0.0625f;  // q4_0 quants come as 16 (n - 8)
    const int t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[i] *= t & 1 ? 65536.0f * Q : Q;
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 1);  // the high digit's lane
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = c * T + (t >> 1);
      if (!(t & 1) && i < cnt) put(i, acc[2 * c], acc[2 * c + 1]);
    }
  }
};

// ------------------------------------------------------------- gate and up
// The compute warps leave a unit's sums (per split) in one of two buffers and
// go on; three further warps add the splits, form h and round it.
struct UpPart {
  float v[2][MOE_KS][MOE_ENT][72];  // [buffer][split][token][32 gate, 32 up, padding]
};
template <int FMT>
__global__ void __launch_bounds__(UP_THREADS, 1) k_moe_up(MoeArgs a) {
  extern __shared__ __align__(128) uint8_t up_smem[];
  __shared__ __align__(8) Pipe pipe;
  constexpr int SG = slab_groups<FMT>(), GB = grp_bytes<FMT>();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) pipe.init();
  uint8_t* const table = up_smem + ring_bytes<FMT>() + sizeof(UpPart);
  clear_table(table, a);
  pdl_wait();
  pdl_trigger();
  UpPart& part = *reinterpret_cast<UpPart*>(up_smem + ring_bytes<FMT>());
  const Table tb = build_table(table, a);
  const int fc = a.F / 32, kg = groups_of(a.K), fg = groups_of(a.F), ns = (kg + SG - 1) / SG;
  const int units = tb.nent * fc, G = gridDim.x;
  // unit u: entry u / fc, chunk u % fc, stepped without divisions
  struct Pos {
    int u, e, c;
  };
  const int de = G / fc, dc = G - de * fc;
  Pos pos{(int)blockIdx.x, (int)blockIdx.x / fc, (int)blockIdx.x % fc};
  auto step = [&]() {
    pos.u += G;
    pos.e += de;
    pos.c += dc;
    if (pos.c >= fc) {
      pos.c -= fc;
      ++pos.e;
    }
  };
  // its entry and its 32 rows.  An expert's entries take turns at the same
  // rows, so that the second reads them from L2.
  auto unit = [&](int& chunk) {
    const uint32_t en = tb.ent[pos.e];
    chunk = pos.c;
    const int at = (int)(en >> 26), run = tb.run(pos.e);
    if (run == 1) return en;
    const int local = at * fc + pos.c;
    chunk = local / run;
    return tb.ent[pos.e - at + local - chunk * run];
  };
  if (warp == MOE_CW) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      Feed<FMT> feed{pipe, saddr(up_smem)};
      bool ok = true;
      for (; pos.u < units && ok; step()) {
        int chunk;
        const uint32_t en = unit(chunk);
        const uint8_t* src = a.gate_up + ((int64_t)(en & 1023u) * fc + chunk) * kg * (MOE_RT * GB);
        for (int g = 0; g < kg && ok; g += SG) ok = feed.put(src + (int64_t)g * MOE_RT * GB, min(SG, kg - g));
      }
      feed.finish();
    }
  } else if (warp < MOE_CW) {
    // ------------------------------------------------------------- compute
    const int rt = warp % MOE_RT, kq = warp / MOE_RT;
    Work<FMT> w;
    w.clear();
    // the unit whose sums are under way (number j here, entry en) and the slab
    // ahead: slab i of the CTA is split i % 3's, counted on through the units
    const int shift = ns % MOE_KS;
    auto first_slab = [&](int l0) { return l0 >= shift ? l0 - shift : l0 - shift + MOE_KS; };
    int j = 0, l = kq, l0 = kq, al = kq, al0 = kq, chunk;
    Turn turn{kq};
    Pos here = pos;  // `pos` runs ahead
    auto take = [&]() {
      const uint32_t en = unit(chunk);
      const int at = (en >> 10) & 0xFFF;
      w.entry(a.xdig, a.xs, kg, (en >> 22) & 15, lane, [&](int i) { return (int64_t)(tb.sorted[at + i] >> 16); });
    };
    auto peek = [&]() {  // the slab ahead, over units that have none for this split
      typename Work<FMT>::Ahead x;
      bool moved = false;
      while (al >= ns) {
        step();
        if (pos.u >= units) return x;
        al0 = first_slab(al0);
        al = al0;
        moved = true;
      }
      if (moved) take();
      return w.ahead(al * SG, min(SG, kg - al * SG));
    };
    typename Work<FMT>::Ahead now;
    if (pos.u < units) {
      take();
      now = peek();
      w.begin(now);
    }
    while (here.u < units) {
      while (l < ns) {
        al += MOE_KS;
        const auto next = peek();
        if (!warp_wait(saddr(&pipe.full[turn.s]), turn.phase, &pipe.abort_flag)) break;
        w.slab(saddr(up_smem) + turn.s * slab_bytes<FMT>(), rt, now, next, lane);
        __syncwarp();  // every lane has read the stage
        if (lane == 0) mbar_arrive(saddr(&pipe.empty[turn.s]));
        turn.next();
        now = next;
        l += MOE_KS;
      }
      if (l < ns) break;  // gave up
      // this unit's sums
      const int b = j & 1;
      const Pos ran = pos;
      pos = here;
      const uint32_t en = unit(chunk);
      step();
      here = pos;
      pos = ran;
      l0 = first_slab(l0);
      l = l0;
      if (j >= 2 && !warp_wait(saddr(&pipe.pempty[b]), (uint32_t)(j / 2 - 1) & 1u, &pipe.abort_flag)) break;
      w.each((en >> 22) & 15, lane, [&](int i, float gate, float up) {
        float* p = part.v[b][kq][i] + rt * 8 + (lane >> 2);
        p[0] = gate;
        p[32] = up;
      });
      w.clear();
      __syncwarp();
      if (lane == 0) mbar_arrive(saddr(&pipe.pfull[b]));
      ++j;
    }
  } else {
    // -------------------------------------------------------------- finish
    for (int j = 0; pos.u < units; ++j, step()) {
      int hb;  // the unit's block of h
      const uint32_t en = unit(hb);
      const int at = (en >> 10) & 0xFFF, cnt = (en >> 22) & 15, b = j & 1;
      if (!warp_wait(saddr(&pipe.pfull[b]), (uint32_t)(j / 2) & 1u, &pipe.abort_flag)) break;
      for (int i = warp - MOE_CW - 1; i < cnt; i += MOE_EW) {
        float gate = 0.0f, up = 0.0f;
#pragma unroll
        for (int q = 0; q < MOE_KS; ++q) {
          gate += part.v[b][q][i][lane];
          up += part.v[b][q][i][32 + lane];
        }
        const int64_t row = tb.sorted[at + i] & 0xFFFFu;
        const float v = gate / (1.0f + expf(-gate)) * up * tb.w[row];
        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7FFFFFFFu);
        const BlockScale bs = block_scale(m);
        const uint32_t f = fixed_biased(v, bs) ^ 0x808080u;
        uint8_t* dst = a.hdig + (row * fg + (hb >> 2)) * DIG_BYTES + ((lane >> 2) & 3) * 32 +
                       (hb & 3) * 8 + (lane >> 4) * 4 + (lane & 3);
#pragma unroll
        for (int p = 0; p < MOE_DIG; ++p) dst[p * 128] = (uint8_t)(f >> (8 * p));
        if (lane == 0) a.hs[row * fg * 4 + hb] = bs.scale;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(saddr(&pipe.pempty[b]));
    }
  }
}

// -------------------------------------------------------------------- down
// A cluster's CTAs have the same 64 rows of y and share out the entries' slabs,
// entry after entry, cut anywhere; the three splits of a CTA add into a copy of
// the 64 rows each.
template <int FMT>
__global__ void __launch_bounds__(DN_THREADS, 1) k_moe_down(MoeArgs a, int ydt) {
  extern __shared__ __align__(128) uint8_t dn_smem[];
  __shared__ __align__(8) Pipe pipe;
  constexpr int SG = slab_groups<FMT>(), GB = grp_bytes<FMT>(), R = 16 * MOE_RT;
  cg::cluster_group cl = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank(), chunk = blockIdx.x / cs;
  if (threadIdx.x == 0) pipe.init();
  float* ypart = reinterpret_cast<float*>(dn_smem + ring_bytes<FMT>());  // [split][token][64]
  const int yn = a.N * R;
  for (int i = threadIdx.x; i < MOE_KS * yn; i += DN_THREADS) ypart[i] = 0.0f;
  uint8_t* const table = dn_smem + ring_bytes<FMT>() + (size_t)MOE_KS * yn * 4;
  clear_table(table, a);
  // The choices are an earlier grid's writes too: that k_moe_up has waited for
  // them orders nothing for this grid, whose SM may still hold an earlier call's.
  // So nothing global is read before this grid's own wait, and no bounded wait
  // (the producer's for empty stages) counts k_moe_up's time.
  pdl_wait();
  pdl_trigger();
  const Table tb = build_table(table, a);
  const int fg = groups_of(a.F), fs = (fg + SG - 1) / SG, chunks = (a.K + R - 1) / R;
  const int64_t total = (int64_t)tb.nent * fs;
  const int q0 = (int)(total * rank / cs), q1 = (int)(total * (rank + 1) / cs);
  if (warp == MOE_CW) {
    if (lane == 0) {
      Feed<FMT> feed{pipe, saddr(dn_smem)};
      int e = q0 / fs, l = q0 - e * fs;
      for (int q = q0; q < q1; ++q) {
        const uint8_t* src = a.down + (((int64_t)(tb.ent[e] & 1023u) * chunks + chunk) * fg + l * SG) * (MOE_RT * GB);
        if (!feed.put(src, min(SG, fg - l * SG))) break;
        if (++l == fs) {
          l = 0;
          ++e;
        }
      }
      feed.finish();
    }
    __syncwarp();
  } else {
    const int rt = warp % MOE_RT, kq = warp / MOE_RT;
    float* yp = ypart + kq * yn + rt * 16 + (lane >> 2);
    Work<FMT> w;
    w.clear();
    // slab q of entry e (`en`: its tokens), and the slab ahead (al of entry ae)
    int q = q0 + kq, ae = q / fs, al = q - ae * fs;
    Turn turn{kq};
    auto take = [&](uint32_t en) {
      const int at = (en >> 10) & 0xFFF;
      w.entry(a.hdig, a.hs, fg, (en >> 22) & 15, lane, [&](int i) { return (int64_t)(tb.sorted[at + i] & 0xFFFFu); });
    };
    typename Work<FMT>::Ahead now;
    uint32_t en = 0;
    if (q < q1) {
      en = tb.ent[ae];
      take(en);
      now = w.ahead(al * SG, min(SG, fg - al * SG));
      w.begin(now);
    }
    while (q < q1) {
      typename Work<FMT>::Ahead next;
      uint32_t nen = en;
      q += MOE_KS;
      if (q < q1) {
        al += MOE_KS;
        if (al >= fs) {
          do {
            al -= fs;
            ++ae;
          } while (al >= fs);
          nen = tb.ent[ae];
          take(nen);
        }
        next = w.ahead(al * SG, min(SG, fg - al * SG));
      }
      if (!warp_wait(saddr(&pipe.full[turn.s]), turn.phase, &pipe.abort_flag)) break;
      w.slab(saddr(dn_smem) + turn.s * slab_bytes<FMT>(), rt, now, next, lane);
      __syncwarp();  // every lane has read the stage
      if (lane == 0) mbar_arrive(saddr(&pipe.empty[turn.s]));
      turn.next();
      now = next;
      if (nen != en || q >= q1) {  // that was the entry's last slab of this warp
        const int at = (en >> 10) & 0xFFF;
        // tokens of an entry are distinct, and the rows are this warp's own
        w.each((en >> 22) & 15, lane, [&](int k, float lo, float hi) {
          float* p = yp + (tb.sorted[at + k] >> 16) * R;
          p[0] += lo;
          p[8] += hi;
        });
        w.clear();
        __syncwarp();  // the next entry may add to the same token from other lanes
        en = nen;
      }
    }
  }
  cl.sync();
  for (int i = rank * DN_THREADS + threadIdx.x; i < yn; i += cs * DN_THREADS) {
    float v = 0.0f;
    for (int c = 0; c < cs; ++c) {
      const float* p = cl.map_shared_rank(ypart, c) + i;
#pragma unroll
      for (int s = 0; s < MOE_KS; ++s) v += p[s * yn];
    }
    const int n = i / R, row = chunk * R + i % R;
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
// One warp per piece: 16 rows (of one matrix, or 8 of each of two) x 128
// columns of one expert; rows and blocks past the last get zeros.
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
  const int per = q2 ? 8 : 16;  // rows of each matrix in a tile
  const int chunks = (rows + per * MOE_RT - 1) / (per * MOE_RT);
  const int64_t ch = wid / (kg * MOE_RT), e = ch / chunks;
  const int grp = (int)(wid / MOE_RT % kg), rt = (int)(ch % chunks) * MOE_RT + (int)(wid % MOE_RT);
  const bool inside = rt * per < rows;  // rows are a multiple of 32: a tile is inside or past the end
  // rows g and g + 8 of the tile
  const int64_t r0 = e * rows + (inside ? rt * per + g : 0);
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
    if (inside && blk < nb) {
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
  const uint32_t s = inside && blk < nb ? (uint32_t)da[blk] | (uint32_t)db[blk] << 16 : 0u;
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
  o += up(n * kg * DIG_BYTES);
  m.xs = o;
  o += up(n * kg * 16);
  m.hdig = o;
  o += up(n * slots * fg * DIG_BYTES);
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

// Clusters of more than 8 CTAs are opt-in per kernel (and device).
int allow_cluster16(const void* f, const DeviceInfo& dev) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_pair(f, dev.device);
  if (done.count(key)) return OK;
  const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return set_error(ERR_CUDA, "allowing clusters of 16: %s", cudaGetErrorString(e));
  done.insert(key);
  return OK;
}

template <int TN>
size_t route_smem(int E) {
  const int epad = (E + rt_cl<TN>() - 1) / rt_cl<TN>();
  return (size_t)TN * rt_chunk<TN>() * 8 + (size_t)RT_WARPS * epad * TN * 8 + (size_t)E * 12;
}

template <int TN>
int launch_route_n(const MoeArgs& a, RouteArgs& r, bool route, bool prep, const DeviceInfo& dev,
                   cudaStream_t st) {
  constexpr int CL = rt_cl<TN>();
  r.clusters = route ? (a.N + TN - 1) / TN : 0;
  // one warp per token and group, at most two CTAs per SM, in whole clusters
  int pre = 0;
  if (prep) {
    const int64_t warps = (int64_t)a.N * groups_of(a.K);
    pre = (int)std::min<int64_t>((warps + RT_WARPS - 1) / RT_WARPS, 2 * dev.sms);
    pre = (pre + CL - 1) / CL * CL;
  }
  if (int rc = allow_max_smem((const void*)k_moe_route<TN>, dev)) return rc;
  if (CL > 8)
    if (int rc = allow_cluster16((const void*)k_moe_route<TN>, dev)) return rc;
  return launch("k_moe_route", k_moe_route<TN>, dim3(CL * r.clusters + pre), RT_THREADS,
                route ? route_smem<TN>(r.E) : 0, CL, st, a, r);
}

// Routing and / or the fixed-point form of x: one launch.
int launch_route(const MoeArgs& a, RouteArgs r, bool route, bool prep, const DeviceInfo& dev,
                 cudaStream_t st) {
  // up to 32 tokens two to a cluster (latency counts: the clusters run side by
  // side), above that sixteen on matrix instructions (512 tokens, 256 experts of
  // 4096 columns: 8 tokens a cluster on DFMA 230 us, now 60)
  if (a.N == 1) return launch_route_n<1>(a, r, route, prep, dev, st);
  if (a.N <= 32) return launch_route_n<2>(a, r, route, prep, dev, st);
  r.clusters = route ? (a.N + RM_TN - 1) / RM_TN : 0;
  int pre = prep ? (int)std::min<int64_t>(((int64_t)a.N * groups_of(a.K) + RT_WARPS - 1) / RT_WARPS, 2 * dev.sms) : 0;
  pre = (pre + RM_CL - 1) / RM_CL * RM_CL;
  if (int rc = allow_max_smem((const void*)k_moe_route_many, dev)) return rc;
  const int epad = (r.E + RM_CL - 1) / RM_CL;
  const size_t smem = route ? (size_t)r.E * 24 + (size_t)rm_slices(epad) * epad * RM_TN * 8 : 0;
  return launch("k_moe_route", k_moe_route_many, dim3(RM_CL * r.clusters + pre), RT_THREADS, smem, RM_CL, st, a, r);
}

template <int FMT>
size_t up_smem(int E, int P, int max_ent) {
  return (size_t)ring_bytes<FMT>() + sizeof(UpPart) + table_bytes(E, P, max_ent);
}
template <int FMT>
size_t dn_smem(int E, int P, int max_ent, int N) {
  return (size_t)ring_bytes<FMT>() + (size_t)MOE_KS * N * 16 * MOE_RT * 4 + table_bytes(E, P, max_ent);
}

template <int FMT>
int launch_up(const MoeArgs& a, const DeviceInfo& dev, cudaStream_t st) {
  if (int rc = allow_max_smem((const void*)k_moe_up<FMT>, dev)) return rc;
  const size_t smem = up_smem<FMT>(a.E, a.N * a.slots, a.max_ent);
  const int64_t units = (int64_t)a.max_ent * (a.F / 32);
  const dim3 grid((unsigned)std::min<int64_t>(units, dev.sms));
  return launch("k_moe_up", k_moe_up<FMT>, grid, UP_THREADS, smem, 0, st, a);
}

template <int FMT>
int launch_down(const MoeArgs& a, int ydt, const DeviceInfo& dev, cudaStream_t st) {
  if (int rc = allow_max_smem((const void*)k_moe_down<FMT>, dev)) return rc;
  const size_t smem = dn_smem<FMT>(a.E, a.N * a.slots, a.max_ent, a.N);
  const int chunks = (a.K + 16 * MOE_RT - 1) / (16 * MOE_RT);
  // CTAs that share 64 rows: as many as leaves every cluster resident at once
  // (one CTA per SM; a GPC's SMs do not divide by every size: 23 clusters of 6
  // took two turns)
  int cs = MOE_DOWN_CL;
  while (cs > 1) {
    int most = 0;
    if (int rc = active_clusters((const void*)k_moe_down<FMT>, dev, DN_THREADS, smem, cs, &most)) return rc;
    if (chunks <= most) break;
    --cs;
  }
  return launch("k_moe_down", k_moe_down<FMT>, dim3(chunks * cs), DN_THREADS, smem, cs, st, a, ydt);
}

}  // namespace

size_t moe_tiles_bytes(int fmt, int64_t E, int64_t rows, int64_t cols) {
  const size_t gb = fmt == 8 ? grp_bytes<8>() : grp_bytes<4>();
  return (size_t)E * ((rows + 63) / 64 * MOE_RT) * groups_of(cols) * gb;
}

int moe_tile(int fmt, const void* q, const void* d, const void* q2, const void* d2, int64_t E,
             int64_t rows, int64_t cols, void* out, cudaStream_t st) {
  const int64_t groups = E * (((q2 ? 2 * rows : rows) + 63) / 64 * MOE_RT) * groups_of(cols);
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
  // tokens of a pass: 64, or fewer where many experts or choices leave too
  // little shared memory for the entries (1024 experts with 32 choices: 32)
  int nt = MOE_NT;
  auto ents = [&](int n) { return std::min(m.E, n * slots) + n * slots / MOE_ENT; };
  while (nt > 1 && std::max(up_smem<4>(m.E, nt * slots, ents(nt)),
                            dn_smem<4>(m.E, nt * slots, ents(nt), nt)) + 1024 > (size_t)dev.smem_optin)
    nt /= 2;
  for (int64_t n0 = 0; n0 < N; n0 += nt) {
    MoeArgs a = {};
    a.x = static_cast<const uint8_t*>(x) + n0 * ldx * xb;
    a.ldx = ldx;
    a.xdt = xdt;
    a.N = (int)std::min<int64_t>(nt, N - n0);
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
    a.max_ent = ents(a.N);  // every entry but an expert's last is full
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
    if (int rc = m.fmt_down == 8 ? launch_down<8>(a, xdt, dev, st) : launch_down<4>(a, xdt, dev, st)) return rc;
  }
  return OK;
}

int set_moe_spin_limit(long long cycles) {
  const cudaError_t e = cudaMemcpyToSymbol(g_moe_spin_limit, &cycles, sizeof(cycles));
  if (e == cudaSuccess) return OK;
  return set_error(ERR_CUDA, "setting the wait limit: %s", cudaGetErrorString(e));
}

int read_moe_error(int clear, cudaStream_t st, int* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_moe_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess)
    return set_error(ERR_CUDA, "reading the device error word: %s", cudaGetErrorString(e));
  if (clear && v) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_moe_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess)
      return set_error(ERR_CUDA, "clearing the device error word: %s", cudaGetErrorString(e));
  }
  *out = v;
  return OK;
}

}  // namespace qg
