// Internal (C++) interfaces between the kernel files and the C ABI in capi.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <mutex>

namespace qg {

// Shared-memory budget for the staged activation tile of the GEMV kernels.
// A whole x of K <= 16384 floats (or N*K floats up to this size) is staged
// once per CTA; larger batches are staged in K tiles.
constexpr size_t kXStageBytes = 64 * 1024;

struct DeviceInfo {
  int device = 0;
  int sms = 0;
  int smem_optin = 0;  // max dynamic shared memory per block (opt-in)
  int cc_major = 0, cc_minor = 0;
  int l2_bytes = 0;
};

// Cached per device; fills `out` for the current device.
int current_device_info(DeviceInfo& out);

// Lets `func` use the device's opt-in shared-memory maximum (once per device).
int allow_max_smem(const void* func, const DeviceInfo& dev);

// Resident blocks per SM of `func` (cached per device, block size and smem).
int occupancy(const void* func, const DeviceInfo& dev, int threads, size_t smem, int* out);

// Clusters of `cs` blocks of `func` that are resident at once with `smem` bytes
// each, of which one block fits an SM (cached per device and cluster size).
int active_clusters(const void* func, const DeviceInfo& dev, int threads, size_t smem, int cs, int* out);

// All-gather fused into the single-column GEMV (one process per GPU): the
// kernel also stores its rows into the other ranks' y buffers (peer
// pointers) and the CTA that finishes last adds 1 to every rank's counter
// sig_out[k]; with sig_in set, the kernel first waits (bounded) until the
// counter of its input reaches (*tok + 1) * nranks.
constexpr int kMaxRanks = 8;
struct FuseArgs {
  float* peer_y[kMaxRanks] = {};
  unsigned* sig_out[kMaxRanks] = {};
  unsigned* cta_count = nullptr;
  const unsigned* sig_in = nullptr;
  const unsigned* tok = nullptr;
  int npeer = 0, nranks = 0;
};

struct GemvCall {
  const void* q = nullptr;  // SoA quant plane, or AoS blocks
  const void* d = nullptr;  // SoA scale plane (fp16 bits); unused for AoS
  const float* x = nullptr;
  float* y = nullptr;
  int64_t M = 0, K = 0;
  int N = 1;
  int64_t ldx = 0, ldy = 0;
  int grid_override = 0;  // >0: force the grid size (tuning / tests)
  void* ws = nullptr;     // workspace of the tensor-core batch kernel
  size_t ws_bytes = 0;
  FuseArgs f;             // fused all-gather (f.nranks == 0: none)
  int act = 0;            // activations: 0 exact (fixed-point planes), 1 q8_1 (opt-in)
  bool no_tc = false;     // batched SoA: keep to the mma.sync kernel (fixed workspace)
};

int gemv_soa(int fmt, const GemvCall& c, cudaStream_t st);
int gemv_soa_variant(int fmt, int variant, const GemvCall& c, cudaStream_t st);
// TMA-fed single-column kernel; returns -1 when the shape is not eligible.
int gemv_soa_tma(int fmt, const GemvCall& c, cudaStream_t st);
bool tma_eligible(const GemvCall& c);
// mode 0: fp32 unpack + FFMA2; mode 1: fixed-point x planes + dp4a.
int gemv_soa_tma_mode(int fmt, int mode, const GemvCall& c, cudaStream_t st);
// GGUF-layout blocks on the TMA path; -1 when the shape is not eligible.
int gemv_aos_tma(int fmt, const GemvCall& c, cudaStream_t st);
// Two columns (N == 2) on the TMA path in one launch, SoA planes or GGUF
// blocks (exact activations; x columns 16-byte aligned); -1 when the call is
// not taken (tma_pair_taken: q4_0 planes and GGUF blocks).  Needs no
// workspace.
bool tma_pair_eligible(const GemvCall& c);
bool tma_pair_taken(int fmt, bool aos, const GemvCall& c);
int gemv_tma_pair(int fmt, bool aos, const GemvCall& c, cudaStream_t st);
int read_device_error(int clear, cudaStream_t st, int* out);
// Persistent decode stack: a sequence of single-column SoA GEMVs in one
// cooperative launch (GEMV j reads GEMV j-1's output).  Outputs are 8-byte
// slots (fp32 bits | tag << 32).  With P ranks (one GPU each) every GEMV's
// rows are also stored into the other ranks' slots (peer_y, rank order
// without this rank).
struct StackCall {
  const void* q;
  const void* d;
  const float* x;           // GEMV 0's input floats
  unsigned long long* y;    // this GEMV's output slots on this rank (M_total)
  int64_t r0, M, M_total, K;
  unsigned long long* peer_y[kMaxRanks - 1] = {};
};
struct StackRanks {
  int nranks = 1, rank = 0;
};
int stack_create(int fmt, const StackCall* calls, int n, const StackRanks* ranks, void** out);
int stack_run(void* handle, cudaStream_t st);
int stack_reset(void* handle, cudaStream_t st);
int stack_destroy(void* handle);
// End of a token of fused calls: signal every rank's done[k], wait (bounded)
// until done_local reaches (*tok + 1) * nranks, then advance *tok.
int token_fence(unsigned* const* done, int nranks, const unsigned* done_local, unsigned* tok,
                cudaStream_t st);
// Tensor-core kernel for 2..16 columns (needs c.ws); -1 when not eligible.
int gemv_soa_mma(int fmt, const GemvCall& c, cudaStream_t st);
bool mma_eligible(const GemvCall& c);
size_t mma_workspace_bytes(int64_t K, int N);
int read_mma_error(int clear, cudaStream_t st, int* out);
// Limits (clock64 cycles) of the bounded waits in the kernels of gemv_tma.cu
// and gemv_mma.cu, on the current device.
int set_spin_limit(long long cycles);
int set_mma_spin_limit(long long cycles);
constexpr long long kDefaultSpinLimit = 2000000000LL;  // ~1 s at ~2 GHz
// Tile counters handed out on `device` so far (one per stream that launched,
// one per captured launch; never returned) and the pool's size.
int tile_counters_used(int device);
int tile_counters_capacity();
// Batch tiles: the weights re-laid for the tensor-core kernel (one contiguous
// block per 16 rows x 512 columns); any K % 32 == 0.
size_t tiled_bytes(int fmt, int64_t M, int64_t K);
int tile_weights(int fmt, bool aos, const void* q, const void* d, int64_t M, int64_t K,
                 void* out, cudaStream_t st);
int gemv_tiled(int fmt, const GemvCall& c, cudaStream_t st);  // c.q = tiles, 1..16 columns
// tc tiles and the tcgen05 batch kernel (gemv_tc.cu), q8_0 (fmt 8) and q4_0
// (fmt 4): 1..16 columns per call; the workspace bound holds for every column
// count and both formats on a device with `sms` SMs.
size_t tc_tiles_bytes(int fmt, int64_t M, int64_t K);
size_t tc_workspace_bytes(int64_t M, int64_t K, int sms);
int tile_weights_tc(int fmt, bool aos, const void* q, const void* d, int64_t M, int64_t K,
                    void* out, cudaStream_t st);
int gemv_tc(int fmt, const void* tiles, int64_t M, int64_t K, const float* x, int64_t ldx,
            float* y, int64_t ldy, int N, void* ws, size_t ws_bytes, cudaStream_t st);
// The same kernel streaming SoA planes through 2-D tensor copies (no
// re-layout): K % 256 == 0, q and d 16-byte aligned; -1 when not eligible or
// when c.ws_bytes is below tc_soa_workspace_bytes.
int gemv_soa_tc(int fmt, const GemvCall& c, cudaStream_t st);
size_t tc_soa_workspace_bytes(int64_t M, int64_t K, int N, int sms);
// A 2-D tensor map (uint8 or uint16 elements; inner dimension contiguous).
int encode_tensor_2d(CUtensorMap* map, bool u16, const void* base, uint64_t inner, uint64_t outer,
                     uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, bool swizzle128);
int set_tc_spin_limit(long long cycles);
int read_tc_error(int clear, cudaStream_t st, int* out);
// Workspace cached per (device, stream) for callers that pass none; grows on
// demand (cudaMalloc, outside stream capture only).  `hold` keeps it for the
// caller until its launches are enqueued: another thread's call on the stream
// waits for that, so that its launches do not come between them (they would
// overwrite what this call's launches pass on) and do not free the buffer.
using WorkspaceHold = std::unique_lock<std::mutex>;
int stream_workspace(cudaStream_t st, size_t bytes, void** out, WorkspaceHold& hold);
// The fixed per-device workspace of qgemv_soa_static_ws (static_ws.cu).
constexpr size_t kStaticWsBytes = (size_t)2 << 20;
int static_workspace(void** out, size_t* bytes);
int release_workspaces();
int soa_variant_count();
const char* soa_variant_name(int v);
int gemv_aos(int fmt, const GemvCall& c, cudaStream_t st);
int fill_zero_rows(float* y, int64_t M, int N, int64_t ldy, cudaStream_t st);

// Quantizers: W fp32 [M][ldw] -> SoA planes (q, d) or AoS blocks.
int quantize(int fmt, const float* w, int64_t M, int64_t K, int64_t ldw, void* q, void* d,
             void* aos, cudaStream_t st);
int dequant(int fmt, const void* q, const void* d, float* w, int64_t M, int64_t K,
            cudaStream_t st);
int repack(int fmt, int to_soa, const void* aos, void* q, void* d, int64_t M, int64_t K,
           cudaStream_t st);

// Roof probes.
int roof_stream_read(const void* buf, size_t bytes, uint32_t* sink, int blocks_per_sm,
                     cudaStream_t st);
int roof_bulk_read(const void* buf, size_t bytes, uint32_t* sink, int* status,
                   cudaStream_t st);

// Mixture of experts (moe.cu).  A pass takes up to kMoeTokens tokens; longer
// calls are split.  dtypes: 0 fp32, 1 bf16, 2 fp16.
constexpr int kMoeTokens = 64;
constexpr int kMoeSlots = 32;     // choices per token, the shared experts among them
constexpr int kMoeExperts = 1024;
constexpr int64_t kMoeMaxDim = (int64_t)1 << 20;  // hidden and inner size
struct MoeRoute {
  const void* w = nullptr;  // router [E][ldw]
  int wdt = 0;
  int64_t ldw = 0;
  const float* bias = nullptr;  // [E], added to the scores for the choice only
  int E = 0, k = 0, scoring = 0, normalize = 1;  // scoring: 0 softmax, 1 sigmoid
  float scale = 1.0f;
};
struct MoeExperts {
  int fmt = 0, fmt_down = 0;  // 8 or 4: gate and up; down
  int E = 0;                  // experts, the shared ones among them
  int64_t K = 0, F = 0;
  const void* gate_up = nullptr;
  const void* down = nullptr;
};
size_t moe_tiles_bytes(int fmt, int64_t E, int64_t rows, int64_t cols);
int moe_tile(int fmt, const void* q, const void* d, const void* q2, const void* d2, int64_t E,
             int64_t rows, int64_t cols, void* out, cudaStream_t st);
size_t moe_workspace_bytes(int64_t N, int slots, int64_t K, int64_t F);
int moe_route(const MoeRoute& c, const void* x, int xdt, int64_t ldx, int64_t N, int64_t K,
              int* ids, float* weights, cudaStream_t st);
// route == nullptr: ids and weights are the caller's; else they are computed.
int moe_experts(const MoeExperts& m, const MoeRoute* route, const void* x, int xdt, int64_t ldx,
                const int* ids, const float* weights, int slots, int64_t N, void* y, int64_t ldy,
                void* ws, cudaStream_t st);

// int8 products (int8.cu).  dtypes as above.
constexpr int64_t kInt8MaxK = ((int64_t)1 << 17) - 1;  // K * 128 * 128 stays in int32
struct Int8Call {
  const void* xq = nullptr;  // int8 [N][ldx]
  const float* xs = nullptr;
  int64_t ldx = 0;
  const void* wq = nullptr;  // int8 [M][ldw]
  const float* ws = nullptr;
  int64_t ldw = 0;
  const float* bias = nullptr;
  int64_t N = 0, M = 0, K = 0;
  void* y = nullptr;
  int64_t ldy = 0;
  int ydt = 0;
};
int int8_quantize(const void* x, int xdt, int64_t ldx, int64_t N, int64_t K, void* q, int64_t ldq,
                  float* s, cudaStream_t st);
// early_w: the launch before this one was int8_quantize's on the same stream
// (the weights may be read before it has finished).
int int8_matmul(const Int8Call& c, bool early_w, cudaStream_t st);
int set_moe_spin_limit(long long cycles);
int read_moe_error(int clear, cudaStream_t st, int* out);
int set_i8_spin_limit(long long cycles);
int read_i8_error(int clear, cudaStream_t st, int* out);

}  // namespace qg
