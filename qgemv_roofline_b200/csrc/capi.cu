// C ABI of libqgemv_b200.so (declared in include/qgemv_b200.h): argument
// validation, error reporting and dispatch to the kernel files.
//
// The reference had no error channel: its harness printed and called exit(1)
// on any CUDA error (src/bench.cu:19-27) and rejected K % 512 != 0
// (src/bench.cu:259).  Here every entry point validates first, returns a
// status code, keeps a per-thread message, and accepts any K % 32 == 0.
#include "qgemv_b200.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <map>
#include <set>
#include <thread>
#include <tuple>
#include <utility>
#include <vector>

#include "qgemv_common.cuh"
#include "qgemv_internal.h"

namespace qg {

static thread_local char g_err[512] = "";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return OK;
}

namespace {
constexpr int kMaxDevices = 64;
std::mutex g_mu;
DeviceInfo g_dev[kMaxDevices];
bool g_dev_ok[kMaxDevices] = {};
std::set<std::pair<const void*, int>> g_smem_set;
struct OccKey {
  const void* f;
  int dev, threads;
  size_t smem;
  bool operator<(const OccKey& o) const {
    return f != o.f ? f < o.f : dev != o.dev ? dev < o.dev
         : threads != o.threads ? threads < o.threads : smem < o.smem;
  }
};
std::map<OccKey, int> g_occ;
}  // namespace

int current_device_info(DeviceInfo& out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) return set_error(ERR_UNSUPPORTED, "device %d", dev);
  std::lock_guard<std::mutex> lk(g_mu);
  if (!g_dev_ok[dev]) {
    DeviceInfo d;
    d.device = dev;
    if ((e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev)) ||
        (e = cudaDeviceGetAttribute(&d.smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev)) ||
        (e = cudaDeviceGetAttribute(&d.cc_major, cudaDevAttrComputeCapabilityMajor, dev)) ||
        (e = cudaDeviceGetAttribute(&d.cc_minor, cudaDevAttrComputeCapabilityMinor, dev)) ||
        (e = cudaDeviceGetAttribute(&d.l2_bytes, cudaDevAttrL2CacheSize, dev)))
      return set_error(ERR_CUDA, "cudaDeviceGetAttribute: %s", cudaGetErrorString(e));
    if (d.cc_major != 10 || d.cc_minor != 0)
      return set_error(ERR_UNSUPPORTED,
                       "device %d is sm_%d%d; this library is built for sm_100a (B200) only", dev,
                       d.cc_major, d.cc_minor);
    g_dev[dev] = d;
    g_dev_ok[dev] = true;
  }
  out = g_dev[dev];
  return OK;
}

int allow_max_smem(const void* func, const DeviceInfo& dev) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto key = std::make_pair(func, dev.device);
  if (g_smem_set.count(key)) return OK;
  // dynamic + static shared memory must stay within the opt-in maximum
  cudaFuncAttributes fa;
  cudaError_t e = cudaFuncGetAttributes(&fa, func);
  if (e != cudaSuccess)
    return set_error(ERR_CUDA, "cudaFuncGetAttributes: %s", cudaGetErrorString(e));
  e = cudaFuncSetAttribute(func, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           dev.smem_optin - (int)fa.sharedSizeBytes);
  if (e != cudaSuccess)
    return set_error(ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  g_smem_set.insert(key);
  return OK;
}

int occupancy(const void* func, const DeviceInfo& dev, int threads, size_t smem, int* out) {
  const OccKey key{func, dev.device, threads, smem};
  {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_occ.find(key);
    if (it != g_occ.end()) {
      *out = it->second;
      return OK;
    }
  }
  int occ = 0;
  const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, func, threads, smem);
  if (e != cudaSuccess || occ < 1)
    return set_error(ERR_CUDA, "occupancy query failed (%s, %d blocks)", cudaGetErrorString(e), occ);
  std::lock_guard<std::mutex> lk(g_mu);
  g_occ[key] = occ;
  *out = occ;
  return OK;
}

int active_clusters(const void* func, const DeviceInfo& dev, int threads, size_t smem, int cs, int* out) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, int>, int> known;
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_tuple(func, dev.device, cs);
  const auto it = known.find(key);
  if (it != known.end()) {
    *out = it->second;
    return OK;
  }
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cs);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, func, &cfg);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(ERR_CUDA, "resident clusters of %d: %s", cs, cudaGetErrorString(e));
  }
  *out = known[key] = n;
  return OK;
}

namespace {

constexpr int64_t kMaxDim = (int64_t)1 << 31;

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) != 0; }

int check_fmt(int format) {
  if (format != 8 && format != 4)
    return set_error(ERR_ARG, "format must be QGEMV_Q8_0 (8) or QGEMV_Q4_0 (4), got %d", format);
  return OK;
}

int check_mk(int64_t M, int64_t K) {
  if (M < 0 || K < 0) return set_error(ERR_SHAPE, "negative shape M=%lld K=%lld", (long long)M, (long long)K);
  if (K % QK) return set_error(ERR_SHAPE, "K=%lld is not a multiple of 32", (long long)K);
  if (M >= kMaxDim || K >= kMaxDim)
    return set_error(ERR_UNSUPPORTED, "M and K must be below 2^31 (M=%lld K=%lld)", (long long)M,
                     (long long)K);
  return OK;
}

// Workspace of a batched SoA call: the tcgen05 kernel's (when it may run) or
// the mma.sync kernel's, whichever is larger (0 when neither runs).
size_t soa_batch_workspace(const GemvCall& probe, bool allow_tc) {
  if (!mma_eligible(probe)) return 0;
  size_t need = mma_workspace_bytes(probe.K, probe.N);
  DeviceInfo dev;
  if (allow_tc && current_device_info(dev) == OK)
    need = std::max(need, tc_soa_workspace_bytes(probe.M, probe.K, probe.N, dev.sms));
  return need;
}

int gemv_entry(int fmt, bool aos, const void* q, const void* d, const float* x, float* y,
               int64_t M, int64_t K, int32_t ncols, int64_t ldx, int64_t ldy, void* stream,
               void* ws = nullptr, size_t ws_bytes = 0, bool caller_ws = false,
               bool allow_tc = true) {
  if (int rc = check_mk(M, K)) return rc;
  if (ncols < 0) return set_error(ERR_SHAPE, "ncols=%d is negative", ncols);
  if (M == 0 || ncols == 0) return OK;
  if (!y || (K > 0 && !x)) return set_error(ERR_NULL, "x and y must not be NULL");
  if (K > 0 && (!q || (!aos && !d)))
    return set_error(ERR_NULL, aos ? "blocks must not be NULL" : "q and d must not be NULL");
  if (ncols > 1 && ldx < K)
    return set_error(ERR_SHAPE, "ldx=%lld < K=%lld", (long long)ldx, (long long)K);
  if (ncols > 1 && ldy < M)
    return set_error(ERR_SHAPE, "ldy=%lld < M=%lld", (long long)ldy, (long long)M);
  if (ncols == 1) {
    ldx = K;
    ldy = M;
  }
  if (K > 0 && misaligned(q, 16))
    return set_error(ERR_ALIGN, aos ? "blocks must be 16-byte aligned" : "q must be 16-byte aligned");
  if (!aos && K > 0 && misaligned(d, 2)) return set_error(ERR_ALIGN, "d must be 2-byte aligned");
  if (misaligned(x, 4) || misaligned(y, 4))
    return set_error(ERR_ALIGN, "x and y must be 4-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) return fill_zero_rows(y, M, ncols, ldy, st);
  GemvCall c;
  c.q = q;
  c.d = d;
  c.x = x;
  c.y = y;
  c.M = M;
  c.K = K;
  c.N = ncols;
  c.ldx = ldx;
  c.ldy = ldy;
  c.no_tc = !allow_tc;
  WorkspaceHold hold;
  if (!aos) {
    // the tensor-core batch kernels need a workspace: the caller's, or one
    // cached for this stream
    // (two columns on the TMA path need none)
    GemvCall probe = c;
    probe.N = std::min(ncols, 16);
    if (probe.N >= 2 && mma_eligible(probe) && !tma_pair_taken(fmt, false, c)) {
      const size_t need = soa_batch_workspace(probe, allow_tc);
      if (caller_ws) {
        if (!ws || ws_bytes < need)
          return set_error(ERR_ARG, "this call needs a workspace of %zu bytes, got %zu", need,
                           ws_bytes);
        if (misaligned(ws, 16)) return set_error(ERR_ALIGN, "workspace must be 16-byte aligned");
      } else if (int rc = stream_workspace(st, need, &ws, hold)) {
        return rc;
      } else {
        ws_bytes = need;
      }
      c.ws = ws;
      c.ws_bytes = ws_bytes;
    }
  }
  return aos ? gemv_aos(fmt, c, st) : gemv_soa(fmt, c, st);
}

// Per-(device, stream) workspaces of the plain entry points.  g_ws_mu guards
// the map, whose entries stay; an entry's own mutex its buffer, and is never
// held while g_ws_mu is asked for.  The per-thread default stream has one
// handle for every thread's stream, hence the thread.
struct StreamWorkspace {
  std::mutex mu;
  void* p = nullptr;
  size_t bytes = 0;
};
std::mutex g_ws_mu;
std::map<std::tuple<int, cudaStream_t, std::thread::id>, StreamWorkspace> g_ws;

}  // namespace

int stream_workspace(cudaStream_t st, size_t bytes, void** out, WorkspaceHold& hold) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error(ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
  const std::thread::id thread = st == cudaStreamPerThread ? std::this_thread::get_id() : std::thread::id();
  StreamWorkspace* slot;
  {
    std::lock_guard<std::mutex> lk(g_ws_mu);
    slot = &g_ws[std::make_tuple(dev, st, thread)];
  }
  WorkspaceHold own(slot->mu);
  if (slot->p && slot->bytes >= bytes) {
    *out = slot->p;
    hold = std::move(own);
    return OK;
  }
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  e = cudaStreamIsCapturing(st, &cs);
  if (e != cudaSuccess || cs != cudaStreamCaptureStatusNone)
    return set_error(ERR_UNSUPPORTED,
                     "a batched call on this stream needs a %zu-byte workspace, which cannot be "
                     "allocated during stream capture: make one uncaptured call of this shape "
                     "on the stream first, or pass a workspace (qgemv_soa_ws)",
                     bytes);
  const size_t grow = std::max(bytes, slot->bytes * 2);
  if (slot->p) {
    // the old buffer may still be read by work queued on this stream
    if ((e = cudaStreamSynchronize(st)) != cudaSuccess || (e = cudaFree(slot->p)) != cudaSuccess)
      return set_error(ERR_CUDA, "releasing the stream workspace: %s", cudaGetErrorString(e));
    slot->p = nullptr;
    slot->bytes = 0;
  }
  void* p = nullptr;
  if ((e = cudaMalloc(&p, grow)) != cudaSuccess)
    return set_error(ERR_CUDA, "allocating a %zu-byte stream workspace: %s", grow,
                     cudaGetErrorString(e));
  slot->p = p;
  slot->bytes = grow;
  *out = p;
  hold = std::move(own);
  return OK;
}

int release_workspaces() {
  std::lock_guard<std::mutex> lk(g_ws_mu);
  int rc = OK;
  for (auto& kv : g_ws) {
    WorkspaceHold own(kv.second.mu);  // a call under way has enqueued its launches
    if (!kv.second.p) continue;
    int cur = 0;
    cudaGetDevice(&cur);
    cudaSetDevice(std::get<0>(kv.first));
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaFree(kv.second.p);
    kv.second.p = nullptr;
    kv.second.bytes = 0;
    cudaSetDevice(cur);
    if (e != cudaSuccess && rc == OK)
      rc = set_error(ERR_CUDA, "releasing a stream workspace: %s", cudaGetErrorString(e));
  }
  return rc;
}

namespace {

}  // namespace
}  // namespace qg

using namespace qg;

extern "C" {

QGEMV_API int qgemv_version(void) { return 100; }

QGEMV_API const char* qgemv_last_error(void) { return g_err; }

QGEMV_API const char* qgemv_status_string(int status) {
  switch (status) {
    case QGEMV_OK: return "QGEMV_OK";
    case QGEMV_ERR_NULL: return "QGEMV_ERR_NULL";
    case QGEMV_ERR_SHAPE: return "QGEMV_ERR_SHAPE";
    case QGEMV_ERR_ALIGN: return "QGEMV_ERR_ALIGN";
    case QGEMV_ERR_CUDA: return "QGEMV_ERR_CUDA";
    case QGEMV_ERR_UNSUPPORTED: return "QGEMV_ERR_UNSUPPORTED";
    case QGEMV_ERR_TIMEOUT: return "QGEMV_ERR_TIMEOUT";
    case QGEMV_ERR_ARG: return "QGEMV_ERR_ARG";
    default: return "QGEMV_ERR_UNKNOWN";
  }
}

QGEMV_API int qgemv_device_info_get(int device, qgemv_device_info* out) {
  if (!out) return set_error(ERR_NULL, "out must not be NULL");
  memset(out, 0, sizeof(*out));
  cudaDeviceProp p;
  cudaError_t e = cudaGetDeviceProperties(&p, device);
  if (e != cudaSuccess)
    return set_error(ERR_CUDA, "cudaGetDeviceProperties(%d): %s", device, cudaGetErrorString(e));
  snprintf(out->name, sizeof(out->name), "%s", p.name);
  out->device = device;
  out->cc_major = p.major;
  out->cc_minor = p.minor;
  out->sms = p.multiProcessorCount;
  out->l2_bytes = p.l2CacheSize;
  cudaDeviceGetAttribute(&out->mem_clock_khz, cudaDevAttrMemoryClockRate, device);
  cudaDeviceGetAttribute(&out->bus_width_bits, cudaDevAttrGlobalMemoryBusWidth, device);
  cudaDeviceGetAttribute(&out->sm_clock_khz, cudaDevAttrClockRate, device);
  cudaDeviceGetAttribute(&out->smem_per_block_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin,
                         device);
  out->datasheet_gbps = 2.0 * out->mem_clock_khz * 1e3 * (out->bus_width_bits / 8.0) / 1e9;
  return OK;
}

QGEMV_API int qgemv_q8_0_soa(const void* q, const void* d, const float* x, float* y, int64_t M,
                             int64_t K, int32_t ncols, int64_t ldx, int64_t ldy, void* stream) {
  return gemv_entry(8, false, q, d, x, y, M, K, ncols, ldx, ldy, stream);
}

QGEMV_API int qgemv_q4_0_soa(const void* q, const void* d, const float* x, float* y, int64_t M,
                             int64_t K, int32_t ncols, int64_t ldx, int64_t ldy, void* stream) {
  return gemv_entry(4, false, q, d, x, y, M, K, ncols, ldx, ldy, stream);
}

QGEMV_API int qgemv_soa_variant_count(void) { return soa_variant_count(); }

QGEMV_API const char* qgemv_soa_variant_name(int variant) { return soa_variant_name(variant); }

QGEMV_API int qgemv_soa_variant(int format, int variant, int32_t grid, const void* q,
                                const void* d, const float* x, float* y, int64_t M, int64_t K,
                                void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (grid < 0) return set_error(ERR_ARG, "grid must be >= 0");
  if (M == 0 || K == 0) return set_error(ERR_SHAPE, "variants need M > 0 and K > 0");
  if (!q || !d || !x || !y) return set_error(ERR_NULL, "q, d, x and y must not be NULL");
  if (misaligned(q, 16) || misaligned(d, 2) || misaligned(x, 4) || misaligned(y, 4))
    return set_error(ERR_ALIGN, "q must be 16-byte, d 2-byte, x and y 4-byte aligned");
  GemvCall c;
  c.q = q;
  c.d = d;
  c.x = x;
  c.y = y;
  c.M = M;
  c.K = K;
  c.N = 1;
  c.ldx = K;
  c.ldy = M;
  c.grid_override = grid;
  return gemv_soa_variant(format, variant, c, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_check_device_error(int clear, void* stream) {
  int v = 0, w = 0, t = 0, i = 0, m = 0;
  if (int rc = read_device_error(clear, static_cast<cudaStream_t>(stream), &v)) return rc;
  if (int rc = read_mma_error(clear, static_cast<cudaStream_t>(stream), &w)) return rc;
  if (int rc = read_tc_error(clear, static_cast<cudaStream_t>(stream), &t)) return rc;
  if (int rc = read_i8_error(clear, static_cast<cudaStream_t>(stream), &i)) return rc;
  if (int rc = read_moe_error(clear, static_cast<cudaStream_t>(stream), &m)) return rc;
  if (!v) v = w;
  if (!v) v = t;
  if (!v) v = i;
  if (!v) v = m;
  if (v) return set_error(v, "a kernel reported %s on the device", qgemv_status_string(v));
  return OK;
}

QGEMV_API int qgemv_set_wait_limit(int64_t microseconds) {
  long long cycles = kDefaultSpinLimit;
  if (microseconds > 0) {
    int dev = 0, khz = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&khz, cudaDevAttrClockRate, dev);
    if (e != cudaSuccess) return set_error(ERR_CUDA, "reading the SM clock: %s", cudaGetErrorString(e));
    if (microseconds > (int64_t)1 << 40) return set_error(ERR_ARG, "wait limit too large");
    cycles = (long long)microseconds * (khz > 0 ? khz : 2000000) / 1000;
    if (cycles < 1) cycles = 1;
  }
  if (int rc = set_spin_limit(cycles)) return rc;
  if (int rc = set_mma_spin_limit(cycles)) return rc;
  if (int rc = set_tc_spin_limit(cycles)) return rc;
  if (int rc = set_i8_spin_limit(cycles)) return rc;
  return set_moe_spin_limit(cycles);
}

QGEMV_API int32_t qgemv_tile_counters_used(int device) { return tile_counters_used(device); }

QGEMV_API int32_t qgemv_tile_counters_capacity(void) { return tile_counters_capacity(); }

QGEMV_API size_t qgemv_soa_workspace_bytes(int format, int64_t M, int64_t K, int32_t ncols) {
  if (check_fmt(format) || check_mk(M, K) || ncols < 2 || M == 0) return 0;
  GemvCall probe;
  probe.M = M;
  probe.K = K;
  probe.N = std::min(ncols, 16);
  // alignment is checked per call; assume aligned planes here
  probe.q = reinterpret_cast<const void*>((uintptr_t)256);
  probe.d = probe.q;
  return soa_batch_workspace(probe, true);
}

QGEMV_API int qgemv_soa_ws(int format, const void* q, const void* d, const float* x, float* y,
                           int64_t M, int64_t K, int32_t ncols, int64_t ldx, int64_t ldy,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  return gemv_entry(format, false, q, d, x, y, M, K, ncols, ldx, ldy, stream, workspace,
                    workspace_bytes, true);
}

QGEMV_API int qgemv_release_workspaces(void) { return release_workspaces(); }

QGEMV_API int qgemv_soa_fused(int format, const void* q, const void* d, const float* x, float* y,
                              int64_t M, int64_t K, const qgemv_fuse* fuse, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (!fuse) return set_error(ERR_NULL, "fuse must not be NULL");
  if (fuse->nranks < 1 || fuse->nranks > kMaxRanks || fuse->npeer < 0 ||
      fuse->npeer > kMaxRanks - 1)
    return set_error(ERR_ARG, "nranks must be in [1, %d] and npeer in [0, %d]", kMaxRanks,
                     kMaxRanks - 1);
  if (!fuse->cta_count || !fuse->tok) return set_error(ERR_NULL, "cta_count and tok must be set");
  for (int k = 0; k < fuse->nranks; ++k)
    if (!fuse->sig_out[k]) return set_error(ERR_NULL, "sig_out[%d] is NULL", k);
  for (int k = 0; k < fuse->npeer; ++k)
    if (!fuse->peer_y[k] || misaligned(fuse->peer_y[k], 4))
      return set_error(ERR_ALIGN, "peer_y[%d] must be a 4-byte aligned device pointer", k);
  if (M == 0) return OK;
  if (!q || !d || !x || !y) return set_error(ERR_NULL, "q, d, x and y must not be NULL");
  if (misaligned(q, 16) || misaligned(d, 2) || misaligned(y, 4))
    return set_error(ERR_ALIGN, "q must be 16-byte, d 2-byte and y 4-byte aligned");
  GemvCall c;
  c.q = q;
  c.d = d;
  c.x = x;
  c.y = y;
  c.M = M;
  c.K = K;
  c.N = 1;
  c.ldx = K;
  c.ldy = M;
  if (!tma_eligible(c))
    return set_error(ERR_UNSUPPORTED,
                     "the fused all-gather needs the TMA kernel: K %% 256 == 0, 256 <= K <= 16384, "
                     "x 16-byte aligned");
  for (int k = 0; k < fuse->nranks; ++k) c.f.sig_out[k] = fuse->sig_out[k];
  for (int k = 0; k < fuse->npeer; ++k) c.f.peer_y[k] = fuse->peer_y[k];
  c.f.cta_count = fuse->cta_count;
  c.f.sig_in = fuse->sig_in;
  c.f.tok = fuse->tok;
  c.f.npeer = fuse->npeer;
  c.f.nranks = fuse->nranks;
  return gemv_soa_tma(format, c, static_cast<cudaStream_t>(stream));
}

namespace {
// Single-column GEMV with q8_1 activations (SoA planes or GGUF blocks).
int q81_entry(int format, bool aos, const void* q, const void* d, const float* x, float* y,
              int64_t M, int64_t K, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (M == 0) return OK;
  if (!x || !y || !q || (!aos && !d))
    return set_error(ERR_NULL, aos ? "blocks, x and y must not be NULL"
                                   : "q, d, x and y must not be NULL");
  if (misaligned(q, 16) || (!aos && misaligned(d, 2)) || misaligned(y, 4))
    return set_error(ERR_ALIGN, aos ? "blocks must be 16-byte and y 4-byte aligned"
                                    : "q must be 16-byte, d 2-byte and y 4-byte aligned");
  GemvCall c;
  c.q = q;
  c.d = d;
  c.x = x;
  c.y = y;
  c.M = M;
  c.K = K;
  c.N = 1;
  c.ldx = K;
  c.ldy = M;
  c.act = 1;
  if (!tma_eligible(c))
    return set_error(ERR_UNSUPPORTED,
                     "q8_1 activations run on the TMA kernel only: K %% 256 == 0, "
                     "256 <= K <= 16384, x 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = aos ? gemv_aos_tma(format, c, st) : gemv_soa_tma(format, c, st);
  return rc == -1 ? set_error(ERR_UNSUPPORTED, "no q8_1 kernel configuration fits this shape")
                  : rc;
}
}  // namespace

QGEMV_API int qgemv_soa_q8_1(int format, const void* q, const void* d, const float* x, float* y,
                             int64_t M, int64_t K, void* stream) {
  return q81_entry(format, false, q, d, x, y, M, K, stream);
}

QGEMV_API int qgemv_aos_q8_1(int format, const void* blocks, const float* x, float* y,
                             int64_t M, int64_t K, void* stream) {
  return q81_entry(format, true, blocks, nullptr, x, y, M, K, stream);
}

namespace {
int stack_entry(int format, const qgemv_stack_gemv* gemvs, int32_t n,
                const qgemv_stack_ranks* ranks, void** handle) {
  if (int rc = check_fmt(format)) return rc;
  if (!gemvs || !handle) return set_error(ERR_NULL, "gemvs and handle must not be NULL");
  if (n < 1 || n > 65536) return set_error(ERR_ARG, "n=%d out of range [1, 65536]", n);
  StackRanks rk;
  if (ranks) {
    if (ranks->nranks < 1 || ranks->nranks > kMaxRanks || ranks->rank < 0 ||
        ranks->rank >= ranks->nranks)
      return set_error(ERR_ARG, "nranks must be in [1, %d] and rank in [0, nranks)", kMaxRanks);
    if (ranks->nranks > 1 && !ranks->peer_y)
      return set_error(ERR_NULL, "peer_y must not be NULL with more than one rank");
    rk.nranks = ranks->nranks;
    rk.rank = ranks->rank;
  }
  std::vector<StackCall> calls(n);
  for (int j = 0; j < n; ++j) {
    const qgemv_stack_gemv& g = gemvs[j];
    if (int rc = check_mk(g.M, g.K)) return rc;
    if (!g.q || !g.d || !g.y || (j == 0 && !g.x))
      return set_error(ERR_NULL, "stack GEMV %d: NULL pointer", j);
    StackCall c;
    c.q = g.q;
    c.d = g.d;
    c.x = g.x;
    c.y = reinterpret_cast<unsigned long long*>(g.y);
    c.r0 = g.r0;
    c.M = g.M;
    c.M_total = g.M_total;
    c.K = g.K;
    for (int k = 0; k < rk.nranks - 1; ++k)
      c.peer_y[k] = reinterpret_cast<unsigned long long*>(
          ranks->peer_y[(size_t)j * (rk.nranks - 1) + k]);
    calls[j] = c;
  }
  *handle = nullptr;
  return stack_create(format, calls.data(), n, ranks ? &rk : nullptr, handle);
}
}  // namespace

QGEMV_API int qgemv_stack_create(int format, const qgemv_stack_gemv* gemvs, int32_t n,
                                 void** handle) {
  return stack_entry(format, gemvs, n, nullptr, handle);
}

QGEMV_API int qgemv_stack_create_ranks(int format, const qgemv_stack_gemv* gemvs, int32_t n,
                                       const qgemv_stack_ranks* ranks, void** handle) {
  if (!ranks) return set_error(ERR_NULL, "ranks must not be NULL");
  return stack_entry(format, gemvs, n, ranks, handle);
}

QGEMV_API int qgemv_stack_run(void* handle, void* stream) {
  if (!handle) return set_error(ERR_NULL, "handle must not be NULL");
  return stack_run(handle, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_stack_reset(void* handle, void* stream) {
  if (!handle) return set_error(ERR_NULL, "handle must not be NULL");
  return stack_reset(handle, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_stack_destroy(void* handle) { return stack_destroy(handle); }

QGEMV_API int qgemv_token_fence(unsigned* const* done, int32_t nranks, const unsigned* done_local,
                                unsigned* tok, void* stream) {
  if (nranks < 1 || nranks > kMaxRanks) return set_error(ERR_ARG, "nranks must be in [1, %d]", kMaxRanks);
  if (!done || !done_local || !tok) return set_error(ERR_NULL, "done, done_local and tok must be set");
  for (int k = 0; k < nranks; ++k)
    if (!done[k]) return set_error(ERR_NULL, "done[%d] is NULL", k);
  return token_fence(const_cast<unsigned* const*>(done), nranks, done_local, tok,
                     static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_soa_static_ws(int format, const void* q, const void* d, const float* x,
                                  float* y, int64_t M, int64_t K, int32_t ncols, int64_t ldx,
                                  int64_t ldy, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  void* ws = nullptr;
  size_t ws_bytes = 0;
  GemvCall probe;
  probe.q = q;
  probe.d = d;
  probe.M = M;
  probe.K = K;
  probe.N = std::min(std::max(ncols, 0), 16);
  // the tcgen05 kernel where its workspace fits the array (it grows with M,
  // the column count and the SM count), else the mma.sync kernel
  bool allow_tc = false;
  if (M > 0 && probe.N >= 2 && mma_eligible(probe)) {
    allow_tc = soa_batch_workspace(probe, true) <= kStaticWsBytes;
    const size_t need = soa_batch_workspace(probe, allow_tc);
    if (need > kStaticWsBytes)
      return set_error(ERR_UNSUPPORTED,
                       "this call needs %zu bytes of workspace; the static workspace holds %zu "
                       "(K <= 32256 at 16 columns): use qgemv_soa_ws",
                       need, kStaticWsBytes);
    if (int rc = static_workspace(&ws, &ws_bytes)) return rc;
  }
  return gemv_entry(format, false, q, d, x, y, M, K, ncols, ldx, ldy, stream, ws, ws_bytes, true,
                    allow_tc);
}

QGEMV_API size_t qgemv_tiled_bytes(int format, int64_t M, int64_t K) {
  if (check_fmt(format) || check_mk(M, K)) return 0;
  return tiled_bytes(format, M, K);
}

QGEMV_API int qgemv_tile_weights(int format, int layout, const void* q, const void* d, int64_t M,
                                 int64_t K, void* tiled, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (layout != 0 && layout != 1)
    return set_error(ERR_ARG, "layout must be 0 (SoA planes) or 1 (ggml blocks), got %d", layout);
  if (M == 0 || K == 0) return OK;
  if (!q || !tiled || (layout == 0 && !d))
    return set_error(ERR_NULL, "source and destination must not be NULL");
  if (misaligned(tiled, 16)) return set_error(ERR_ALIGN, "tiles must be 16-byte aligned");
  if (layout == 0 && (misaligned(q, 16) || misaligned(d, 2)))
    return set_error(ERR_ALIGN, "q must be 16-byte and d 2-byte aligned");
  return tile_weights(format, layout == 1, q, d, M, K, tiled, static_cast<cudaStream_t>(stream));
}

QGEMV_API size_t qgemv_tiled_workspace_bytes(int64_t K, int32_t ncols) {
  if (K < 0 || K % QK || ncols < 1) return 0;
  return mma_workspace_bytes(K, ncols);
}

QGEMV_API int qgemv_tiled_gemv(int format, const void* tiled, int64_t M, int64_t K,
                               const float* x, float* y, int32_t ncols, int64_t ldx, int64_t ldy,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (K > ((int64_t)1 << 20))
    return set_error(ERR_UNSUPPORTED, "K=%lld above 2^20 for batch tiles", (long long)K);
  if (ncols < 0) return set_error(ERR_SHAPE, "ncols=%d is negative", ncols);
  if (M == 0 || ncols == 0) return OK;
  if (!y || (K > 0 && (!x || !tiled))) return set_error(ERR_NULL, "tiles, x and y must not be NULL");
  if (ncols > 1 && ldx < K) return set_error(ERR_SHAPE, "ldx=%lld < K=%lld", (long long)ldx, (long long)K);
  if (ncols > 1 && ldy < M) return set_error(ERR_SHAPE, "ldy=%lld < M=%lld", (long long)ldy, (long long)M);
  if (ncols == 1) {
    ldx = K;
    ldy = M;
  }
  if (K > 0 && misaligned(tiled, 16)) return set_error(ERR_ALIGN, "tiles must be 16-byte aligned");
  if (misaligned(x, 4) || misaligned(y, 4)) return set_error(ERR_ALIGN, "x and y must be 4-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) return fill_zero_rows(y, M, ncols, ldy, st);
  const size_t need = mma_workspace_bytes(K, ncols);
  WorkspaceHold hold;
  if (workspace) {
    if (workspace_bytes < need)
      return set_error(ERR_ARG, "this call needs a workspace of %zu bytes, got %zu", need,
                       workspace_bytes);
    if (misaligned(workspace, 16)) return set_error(ERR_ALIGN, "workspace must be 16-byte aligned");
  } else if (int rc = stream_workspace(st, need, &workspace, hold)) {
    return rc;
  } else {
    workspace_bytes = need;
  }
  GemvCall c;
  c.q = tiled;
  c.M = M;
  c.K = K;
  c.ldx = ldx;
  c.ldy = ldy;
  c.ws = workspace;
  c.ws_bytes = workspace_bytes;
  for (int n0 = 0; n0 < ncols; n0 += 16) {
    c.N = std::min(16, ncols - n0);
    c.x = x + (int64_t)n0 * ldx;
    c.y = y + (int64_t)n0 * ldy;
    if (int rc = gemv_tiled(format, c, st)) return rc;
  }
  return OK;
}

QGEMV_API size_t qgemv_tc_bytes(int format, int64_t M, int64_t K) {
  if (check_fmt(format) || check_mk(M, K)) return 0;
  return tc_tiles_bytes(format, M, K);
}

QGEMV_API int qgemv_tc_tile(int format, int layout, const void* q, const void* d, int64_t M,
                            int64_t K, void* tiles, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (layout != 0 && layout != 1)
    return set_error(ERR_ARG, "layout must be 0 (SoA planes) or 1 (ggml blocks), got %d", layout);
  if (M == 0 || K == 0) return OK;
  if (!q || !tiles || (layout == 0 && !d))
    return set_error(ERR_NULL, "source and destination must not be NULL");
  if (misaligned(tiles, 16)) return set_error(ERR_ALIGN, "tiles must be 16-byte aligned");
  if (layout == 0 && (misaligned(q, 16) || misaligned(d, 2)))
    return set_error(ERR_ALIGN, "q must be 16-byte and d 2-byte aligned");
  return tile_weights_tc(format, layout == 1, q, d, M, K, tiles, static_cast<cudaStream_t>(stream));
}

QGEMV_API size_t qgemv_tc_workspace_bytes(int64_t M, int64_t K) {
  if (check_mk(M, K)) return 0;
  DeviceInfo dev;
  if (current_device_info(dev)) return 0;
  return tc_workspace_bytes(M, K, dev.sms);
}

QGEMV_API int qgemv_tc_gemv(int format, const void* tiles, int64_t M, int64_t K, const float* x,
                            float* y, int32_t ncols, int64_t ldx, int64_t ldy, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (K > ((int64_t)1 << 20))
    return set_error(ERR_UNSUPPORTED, "K=%lld above 2^20 for tc tiles", (long long)K);
  if (ncols < 0) return set_error(ERR_SHAPE, "ncols=%d is negative", ncols);
  if (M == 0 || ncols == 0) return OK;
  if (!y || (K > 0 && (!x || !tiles))) return set_error(ERR_NULL, "tiles, x and y must not be NULL");
  if (ncols > 1 && ldx < K) return set_error(ERR_SHAPE, "ldx=%lld < K=%lld", (long long)ldx, (long long)K);
  if (ncols > 1 && ldy < M) return set_error(ERR_SHAPE, "ldy=%lld < M=%lld", (long long)ldy, (long long)M);
  if (ncols == 1) {
    ldx = K;
    ldy = M;
  }
  if (K > 0 && misaligned(tiles, 16)) return set_error(ERR_ALIGN, "tiles must be 16-byte aligned");
  if (misaligned(x, 4) || misaligned(y, 4)) return set_error(ERR_ALIGN, "x and y must be 4-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (K == 0) return fill_zero_rows(y, M, ncols, ldy, st);
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  const size_t need = tc_workspace_bytes(M, K, dev.sms);
  WorkspaceHold hold;
  if (workspace) {
    if (workspace_bytes < need)
      return set_error(ERR_ARG, "this call needs a workspace of %zu bytes, got %zu", need,
                       workspace_bytes);
    if (misaligned(workspace, 16)) return set_error(ERR_ALIGN, "workspace must be 16-byte aligned");
  } else if (int rc = stream_workspace(st, need, &workspace, hold)) {
    return rc;
  } else {
    workspace_bytes = need;
  }
  for (int n0 = 0; n0 < ncols; n0 += 16) {
    const int n = std::min(16, ncols - n0);
    if (int rc = gemv_tc(format, tiles, M, K, x + (int64_t)n0 * ldx, ldx, y + (int64_t)n0 * ldy,
                         ldy, n, workspace, workspace_bytes, st))
      return rc;
  }
  return OK;
}

QGEMV_API size_t qgemv_q8_0_tc_bytes(int64_t M, int64_t K) { return qgemv_tc_bytes(8, M, K); }

QGEMV_API int qgemv_q8_0_tc_tile(int layout, const void* q, const void* d, int64_t M, int64_t K,
                                 void* tiles, void* stream) {
  return qgemv_tc_tile(8, layout, q, d, M, K, tiles, stream);
}

QGEMV_API size_t qgemv_q8_0_tc_workspace_bytes(int64_t M, int64_t K) {
  return qgemv_tc_workspace_bytes(M, K);
}

QGEMV_API int qgemv_q8_0_tc(const void* tiles, int64_t M, int64_t K, const float* x, float* y,
                            int32_t ncols, int64_t ldx, int64_t ldy, void* workspace,
                            size_t workspace_bytes, void* stream) {
  return qgemv_tc_gemv(8, tiles, M, K, x, y, ncols, ldx, ldy, workspace, workspace_bytes, stream);
}

QGEMV_API int qgemv_q8_0_aos(const void* blocks, const float* x, float* y, int64_t M, int64_t K,
                             int32_t ncols, int64_t ldx, int64_t ldy, void* stream) {
  return gemv_entry(8, true, blocks, nullptr, x, y, M, K, ncols, ldx, ldy, stream);
}

QGEMV_API int qgemv_q4_0_aos(const void* blocks, const float* x, float* y, int64_t M, int64_t K,
                             int32_t ncols, int64_t ldx, int64_t ldy, void* stream) {
  return gemv_entry(4, true, blocks, nullptr, x, y, M, K, ncols, ldx, ldy, stream);
}

QGEMV_API int qgemv_quantize_soa(int format, const float* w, int64_t M, int64_t K, int64_t ldw,
                                 void* q, void* d, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (M == 0 || K == 0) return OK;
  if (!w || !q || !d) return set_error(ERR_NULL, "w, q and d must not be NULL");
  if (ldw < K) return set_error(ERR_SHAPE, "ldw=%lld < K=%lld", (long long)ldw, (long long)K);
  if (misaligned(w, 4) || misaligned(d, 2))
    return set_error(ERR_ALIGN, "w must be 4-byte and d 2-byte aligned");
  return quantize(format, w, M, K, ldw, q, d, nullptr, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_quantize_aos(int format, const float* w, int64_t M, int64_t K, int64_t ldw,
                                 void* blocks, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (M == 0 || K == 0) return OK;
  if (!w || !blocks) return set_error(ERR_NULL, "w and blocks must not be NULL");
  if (ldw < K) return set_error(ERR_SHAPE, "ldw=%lld < K=%lld", (long long)ldw, (long long)K);
  if (misaligned(w, 4)) return set_error(ERR_ALIGN, "w must be 4-byte aligned");
  return quantize(format, w, M, K, ldw, nullptr, nullptr, blocks,
                  static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_dequant_soa(int format, const void* q, const void* d, float* w, int64_t M,
                                int64_t K, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (int rc = check_mk(M, K)) return rc;
  if (M == 0 || K == 0) return OK;
  if (!q || !d || !w) return set_error(ERR_NULL, "q, d and w must not be NULL");
  if (misaligned(w, 4) || misaligned(d, 2))
    return set_error(ERR_ALIGN, "w must be 4-byte and d 2-byte aligned");
  return dequant(format, q, d, w, M, K, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_repack(int format, int to_soa, void* blocks, void* q, void* d, int64_t M,
                           int64_t K, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (to_soa != 0 && to_soa != 1) return set_error(ERR_ARG, "to_soa must be 0 or 1");
  if (int rc = check_mk(M, K)) return rc;
  if (M == 0 || K == 0) return OK;
  if (!blocks || !q || !d) return set_error(ERR_NULL, "blocks, q and d must not be NULL");
  if (misaligned(d, 2)) return set_error(ERR_ALIGN, "d must be 2-byte aligned");
  return repack(format, to_soa, blocks, q, d, M, K, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_roof_stream_read(const void* buf, size_t bytes, uint32_t* sink,
                                     int32_t blocks_per_sm, void* stream) {
  if (!buf || !sink) return set_error(ERR_NULL, "buf and sink must not be NULL");
  if (bytes % 16) return set_error(ERR_SHAPE, "bytes must be a multiple of 16");
  if (misaligned(buf, 16) || misaligned(sink, 4))
    return set_error(ERR_ALIGN, "buf must be 16-byte and sink 4-byte aligned");
  if (blocks_per_sm < 1 || blocks_per_sm > 64)
    return set_error(ERR_ARG, "blocks_per_sm must be in [1, 64]");
  return roof_stream_read(buf, bytes, sink, blocks_per_sm, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_roof_bulk_read(const void* buf, size_t bytes, uint32_t* sink, int* status,
                                   void* stream) {
  if (!buf || !sink || !status) return set_error(ERR_NULL, "buf, sink and status must not be NULL");
  if (bytes % 16) return set_error(ERR_SHAPE, "bytes must be a multiple of 16");
  if (misaligned(buf, 16) || misaligned(sink, 4) || misaligned(status, 4))
    return set_error(ERR_ALIGN, "buf must be 16-byte aligned; sink and status 4-byte");
  return roof_bulk_read(buf, bytes, sink, status, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_roof_d2d(void* dst, const void* src, size_t bytes, void* stream) {
  if (!dst || !src) return set_error(ERR_NULL, "dst and src must not be NULL");
  const cudaError_t e =
      cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToDevice, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return set_error(ERR_CUDA, "cudaMemcpyAsync: %s", cudaGetErrorString(e));
  return OK;
}

QGEMV_API size_t qgemv_moe_tiles_bytes(int format, int64_t n_experts, int64_t rows, int64_t cols) {
  if (check_fmt(format) || n_experts < 0 || n_experts > kMoeExperts || rows < 0 || rows % 16 ||
      cols < 0 || cols % QK || rows > kMoeMaxDim * 2 || cols > kMoeMaxDim)
    return 0;
  return moe_tiles_bytes(format, n_experts, rows, cols);
}

QGEMV_API int qgemv_moe_tile(int format, const void* q, const void* d, const void* q2,
                             const void* d2, int64_t n_experts, int64_t rows, int64_t cols,
                             void* out, void* stream) {
  if (int rc = check_fmt(format)) return rc;
  if (n_experts < 0 || n_experts > kMoeExperts)
    return set_error(ERR_ARG, "n_experts=%lld out of range [0, %d]", (long long)n_experts, kMoeExperts);
  if (rows < 0 || cols < 0 || rows % QK || cols % QK)
    return set_error(ERR_SHAPE, "rows=%lld and cols=%lld must be multiples of 32", (long long)rows,
                     (long long)cols);
  if (rows > kMoeMaxDim || cols > kMoeMaxDim)
    return set_error(ERR_UNSUPPORTED, "expert matrices of up to 2^20 rows and columns");
  if (!n_experts || !rows || !cols) return OK;
  if (!q || !d || !out || (q2 && !d2)) return set_error(ERR_NULL, "q, d and out must not be NULL");
  if (misaligned(q, 16) || misaligned(q2, 16) || misaligned(out, 16) || misaligned(d, 2) ||
      misaligned(d2, 2))
    return set_error(ERR_ALIGN, "quants and out must be 16-byte, scales 2-byte aligned");
  return moe_tile(format, q, d, q2, d2, n_experts, rows, cols, out, static_cast<cudaStream_t>(stream));
}

namespace {
// The stream's workspace for a call that brought none.  Refused under capture:
// a graph would keep the buffer's address, which a later, larger call on the
// stream frees, and graphs captured on one stream would share it.
int own_workspace(cudaStream_t st, size_t need, void** ws, WorkspaceHold& hold) {
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  const cudaError_t e = cudaStreamIsCapturing(st, &cs);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(ERR_CUDA, "cudaStreamIsCapturing: %s", cudaGetErrorString(e));
  }
  if (cs != cudaStreamCaptureStatusNone)
    return set_error(ERR_UNSUPPORTED, "a captured call needs a workspace of its own (%zu bytes)", need);
  return stream_workspace(st, need, ws, hold);
}

int check_moe_x(const void* x, int dtype, int64_t ldx, int64_t N, int64_t K) {
  if (dtype < 0 || dtype > 2) return set_error(ERR_ARG, "dtype must be 0, 1 or 2, got %d", dtype);
  if (N < 0 || K < 1) return set_error(ERR_SHAPE, "n_tokens=%lld hidden=%lld", (long long)N, (long long)K);
  if (N >= kMaxDim || K > kMoeMaxDim)
    return set_error(ERR_UNSUPPORTED, "n_tokens must be below 2^31 and hidden at most 2^20");
  if (N == 0) return OK;
  if (!x) return set_error(ERR_NULL, "x must not be NULL");
  if (misaligned(x, dtype == 0 ? 4 : 2)) return set_error(ERR_ALIGN, "x must be aligned to its elements");
  if (ldx < (N > 1 ? K : 0)) return set_error(ERR_SHAPE, "ldx=%lld < hidden=%lld", (long long)ldx, (long long)K);
  return OK;
}

int check_router(const qgemv_moe_router* r, int64_t K, MoeRoute& out) {
  if (!r) return set_error(ERR_NULL, "router must not be NULL");
  if (r->w_dtype < 0 || r->w_dtype > 2)
    return set_error(ERR_ARG, "w_dtype must be 0, 1 or 2, got %d", r->w_dtype);
  if (r->n_experts < 1 || r->n_experts > kMoeExperts)
    return set_error(ERR_ARG, "n_experts=%d out of range [1, %d]", r->n_experts, kMoeExperts);
  if (r->top_k < 1 || r->top_k > r->n_experts || r->top_k > kMoeSlots)
    return set_error(ERR_ARG, "top_k=%d out of range [1, min(%d experts, %d)]", r->top_k, r->n_experts,
                     kMoeSlots);
  if (r->scoring != 0 && r->scoring != 1)
    return set_error(ERR_ARG, "scoring must be 0 (softmax) or 1 (sigmoid), got %d", r->scoring);
  if (!r->w) return set_error(ERR_NULL, "the router's weights must not be NULL");
  if (misaligned(r->w, r->w_dtype == 0 ? 4 : 2) || misaligned(r->bias, 4))
    return set_error(ERR_ALIGN, "the router's weights must be aligned to their elements, its bias to 4 bytes");
  if (r->ldw < (r->n_experts > 1 ? K : 0))
    return set_error(ERR_SHAPE, "ldw=%lld < hidden=%lld", (long long)r->ldw, (long long)K);
  out.w = r->w;
  out.wdt = r->w_dtype;
  out.ldw = r->ldw;
  out.bias = r->bias;
  out.E = r->n_experts;
  out.k = r->top_k;
  out.scoring = r->scoring;
  out.normalize = r->normalize != 0;
  out.scale = r->scale;
  return OK;
}

int moe_entry(const qgemv_expert_set* m, const qgemv_moe_router* router, const void* x, int dtype,
              int64_t ldx, const int32_t* ids, const float* weights, int32_t slots, int64_t N,
              void* y, int64_t ldy, void* ws, size_t ws_bytes, void* stream) {
  if (!m) return set_error(ERR_NULL, "experts must not be NULL");
  if (int rc = check_fmt(m->format)) return rc;
  if (int rc = check_fmt(m->format_down)) return rc;
  if (m->n_experts < 1 || m->n_experts > kMoeExperts || m->n_shared < 0 || m->n_shared > m->n_experts)
    return set_error(ERR_ARG, "n_experts=%d (of them n_shared=%d) out of range [1, %d]", m->n_experts,
                     m->n_shared, kMoeExperts);
  if (m->hidden < QK || m->ffn < QK || m->hidden % QK || m->ffn % QK)
    return set_error(ERR_SHAPE, "hidden=%lld and ffn=%lld must be multiples of 32", (long long)m->hidden,
                     (long long)m->ffn);
  if (m->hidden > kMoeMaxDim || m->ffn > kMoeMaxDim)
    return set_error(ERR_UNSUPPORTED, "hidden and ffn must be at most 2^20");
  if (int rc = check_moe_x(x, dtype, ldx, N, m->hidden)) return rc;
  MoeRoute route;
  if (router) {
    if (int rc = check_router(router, m->hidden, route)) return rc;
    if (router->n_experts != m->n_experts - m->n_shared)
      return set_error(ERR_SHAPE, "the router has %d rows for %d routed experts", router->n_experts,
                       m->n_experts - m->n_shared);
    slots = router->top_k + m->n_shared;
  }
  if (slots < 1 || slots > kMoeSlots)
    return set_error(ERR_ARG, "%d choices per token, out of range [1, %d]", slots, kMoeSlots);
  if (N == 0) return OK;
  if (!y || !m->gate_up || !m->down) return set_error(ERR_NULL, "y and the tiles must not be NULL");
  if (!router && (!ids || !weights)) return set_error(ERR_NULL, "ids and weights must not be NULL");
  if (misaligned(m->gate_up, 16) || misaligned(m->down, 16) || misaligned(y, dtype == 0 ? 4 : 2) ||
      misaligned(ids, 4) || misaligned(weights, 4))
    return set_error(ERR_ALIGN, "tiles must be 16-byte aligned, ids and weights 4-byte, y to its elements");
  if (ldy < (N > 1 ? m->hidden : 0))
    return set_error(ERR_SHAPE, "ldy=%lld < hidden=%lld", (long long)ldy, (long long)m->hidden);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t need = moe_workspace_bytes(N, slots, m->hidden, m->ffn);
  WorkspaceHold hold;
  if (ws) {
    if (ws_bytes < need)
      return set_error(ERR_ARG, "this call needs a workspace of %zu bytes, got %zu", need, ws_bytes);
    if (misaligned(ws, 16)) return set_error(ERR_ALIGN, "workspace must be 16-byte aligned");
  } else if (int rc = own_workspace(st, need, &ws, hold)) {
    return rc;
  }
  MoeExperts e;
  e.fmt = m->format;
  e.fmt_down = m->format_down;
  e.E = m->n_experts;
  e.K = m->hidden;
  e.F = m->ffn;
  e.gate_up = m->gate_up;
  e.down = m->down;
  return moe_experts(e, router ? &route : nullptr, x, dtype, ldx, ids, weights, slots, N, y, ldy, ws, st);
}
}  // namespace

QGEMV_API int qgemv_moe_route(const qgemv_moe_router* router, const void* x, int dtype,
                              int64_t ldx, int64_t n_tokens, int64_t hidden, int32_t* ids,
                              float* weights, void* stream) {
  if (int rc = check_moe_x(x, dtype, ldx, n_tokens, hidden)) return rc;
  MoeRoute r;
  if (int rc = check_router(router, hidden, r)) return rc;
  if (n_tokens == 0) return OK;
  if (!ids || !weights) return set_error(ERR_NULL, "ids and weights must not be NULL");
  if (misaligned(ids, 4) || misaligned(weights, 4))
    return set_error(ERR_ALIGN, "ids and weights must be 4-byte aligned");
  return moe_route(r, x, dtype, ldx, n_tokens, hidden, ids, weights, static_cast<cudaStream_t>(stream));
}

QGEMV_API size_t qgemv_moe_workspace_bytes(int64_t n_tokens, int32_t slots, int64_t hidden,
                                           int64_t ffn) {
  if (n_tokens < 1 || slots < 1 || slots > kMoeSlots || hidden < QK || ffn < QK || hidden % QK ||
      ffn % QK || hidden > kMoeMaxDim || ffn > kMoeMaxDim)
    return 0;
  return moe_workspace_bytes(n_tokens, slots, hidden, ffn);
}

QGEMV_API int qgemv_moe_experts(const qgemv_expert_set* experts, const void* x, int dtype,
                                int64_t ldx, const int32_t* ids, const float* weights,
                                int32_t slots, int64_t n_tokens, void* y, int64_t ldy,
                                void* workspace, size_t workspace_bytes, void* stream) {
  return moe_entry(experts, nullptr, x, dtype, ldx, ids, weights, slots, n_tokens, y, ldy,
                   workspace, workspace_bytes, stream);
}

QGEMV_API int qgemv_moe_layer(const qgemv_expert_set* experts, const qgemv_moe_router* router,
                              const void* x, int dtype, int64_t ldx, int64_t n_tokens, void* y,
                              int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
  if (!router) return set_error(ERR_NULL, "router must not be NULL");
  return moe_entry(experts, router, x, dtype, ldx, nullptr, nullptr, 0, n_tokens, y, ldy,
                   workspace, workspace_bytes, stream);
}

namespace {
int check_int8_rows(const char* what, const void* q, int64_t ld, int64_t rows, int64_t K) {
  if (!q) return set_error(ERR_NULL, "%s must not be NULL", what);
  if (misaligned(q, 16) || (rows > 1 && ld % 16))
    return set_error(ERR_ALIGN, "%s and its rows must be 16-byte aligned", what);
  if (rows > 1 && (ld < K || ld >= ((int64_t)1 << 39)))
    return set_error(ERR_SHAPE, "%s: row stride %lld for %lld columns", what, (long long)ld, (long long)K);
  return OK;
}

int check_int8_sizes(int64_t N, int64_t M, int64_t K) {
  if (N < 0 || M < 0) return set_error(ERR_SHAPE, "negative shape N=%lld M=%lld", (long long)N, (long long)M);
  if (K < 16 || K % 16) return set_error(ERR_SHAPE, "K=%lld is not a positive multiple of 16", (long long)K);
  if (K > kInt8MaxK)
    return set_error(ERR_UNSUPPORTED, "K=%lld: int32 sums are exact up to K=%lld", (long long)K,
                     (long long)kInt8MaxK);
  if (N >= kMaxDim - 512 || M >= kMaxDim - 512)  // tile origins stay in 32 bits
    return set_error(ERR_UNSUPPORTED, "N and M must be below 2^31 - 512 (N=%lld M=%lld)", (long long)N, (long long)M);
  return OK;
}

int int8_entry(const void* xq, const float* xs, int64_t ldx, const void* wq, const float* ws, int64_t ldw,
               const float* bias, int64_t N, int64_t M, int64_t K, void* y, int ydt, int64_t ldy,
               bool early_w, void* stream) {
  if (ydt < 0 || ydt > 2) return set_error(ERR_ARG, "y_dtype must be 0, 1 or 2, got %d", ydt);
  if (int rc = check_int8_sizes(N, M, K)) return rc;
  if (N == 0 || M == 0) return OK;
  if (int rc = check_int8_rows("xq", xq, ldx, N, K)) return rc;
  if (int rc = check_int8_rows("wq", wq, ldw, M, K)) return rc;
  if (!xs || !ws || !y) return set_error(ERR_NULL, "xs, ws and y must not be NULL");
  if (misaligned(xs, 4) || misaligned(ws, 4) || misaligned(bias, 4) || misaligned(y, ydt == 0 ? 4 : 2))
    return set_error(ERR_ALIGN, "scales and bias must be 4-byte aligned, y to its elements");
  if (ldy < (N > 1 ? M : 0)) return set_error(ERR_SHAPE, "ldy=%lld < M=%lld", (long long)ldy, (long long)M);
  Int8Call c;
  c.xq = xq;
  c.xs = xs;
  c.ldx = N > 1 ? ldx : (K + 15) / 16 * 16;
  c.wq = wq;
  c.ws = ws;
  c.ldw = M > 1 ? ldw : (K + 15) / 16 * 16;
  c.bias = bias;
  c.N = N;
  c.M = M;
  c.K = K;
  c.y = y;
  c.ldy = ldy;
  c.ydt = ydt;
  return int8_matmul(c, early_w, static_cast<cudaStream_t>(stream));
}
}  // namespace

QGEMV_API int qgemv_int8_quantize(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t K,
                                  void* q, int64_t ldq, float* scales, void* stream) {
  if (dtype < 0 || dtype > 2) return set_error(ERR_ARG, "dtype must be 0, 1 or 2, got %d", dtype);
  if (rows < 0 || K < 1) return set_error(ERR_SHAPE, "rows=%lld K=%lld", (long long)rows, (long long)K);
  if (rows >= kMaxDim || K >= kMaxDim - 512)  // a row's columns are counted in 32 bits, 256 at a time
    return set_error(ERR_UNSUPPORTED, "rows must be below 2^31 and K below 2^31 - 512 (rows=%lld K=%lld)",
                     (long long)rows, (long long)K);
  if (rows == 0) return OK;
  if (!x || !q || !scales) return set_error(ERR_NULL, "x, q and scales must not be NULL");
  if (misaligned(x, dtype == 0 ? 4 : 2) || misaligned(scales, 4))
    return set_error(ERR_ALIGN, "x must be aligned to its elements, scales to 4 bytes");
  if (rows > 1 && (ldx < K || ldq < K))
    return set_error(ERR_SHAPE, "ldx=%lld and ldq=%lld must be at least K=%lld", (long long)ldx,
                     (long long)ldq, (long long)K);
  return int8_quantize(x, dtype, ldx, rows, K, q, ldq, scales, static_cast<cudaStream_t>(stream));
}

QGEMV_API int qgemv_int8_matmul(const void* xq, const float* xs, int64_t ldx, const void* wq,
                                const float* ws, int64_t ldw, const float* bias, int64_t N,
                                int64_t M, int64_t K, void* y, int y_dtype, int64_t ldy, void* stream) {
  return int8_entry(xq, xs, ldx, wq, ws, ldw, bias, N, M, K, y, y_dtype, ldy, false, stream);
}

QGEMV_API size_t qgemv_int8_linear_workspace_bytes(int64_t N, int64_t K) {
  if (N < 1 || K < 16 || K % 16 || K > kInt8MaxK || N >= kMaxDim) return 0;
  return (size_t)((N + 31) / 32 * 32) * 4 + (size_t)N * K;
}

QGEMV_API int qgemv_int8_linear(const void* x, int dtype, int64_t ldx, const void* wq, const float* ws,
                                int64_t ldw, const float* bias, int64_t N, int64_t M, int64_t K,
                                void* y, int y_dtype, int64_t ldy, void* workspace,
                                size_t workspace_bytes, void* stream) {
  if (dtype < 0 || dtype > 2) return set_error(ERR_ARG, "dtype must be 0, 1 or 2, got %d", dtype);
  if (int rc = check_int8_sizes(N, M, K)) return rc;
  if (N == 0 || M == 0) return OK;
  if (!x) return set_error(ERR_NULL, "x must not be NULL");
  if (misaligned(x, dtype == 0 ? 4 : 2)) return set_error(ERR_ALIGN, "x must be aligned to its elements");
  if (ldx < (N > 1 ? K : 0)) return set_error(ERR_SHAPE, "ldx=%lld < K=%lld", (long long)ldx, (long long)K);
  // everything the product checks, before anything is launched
  if (y_dtype < 0 || y_dtype > 2) return set_error(ERR_ARG, "y_dtype must be 0, 1 or 2, got %d", y_dtype);
  if (int rc = check_int8_rows("wq", wq, ldw, M, K)) return rc;
  if (!ws || !y) return set_error(ERR_NULL, "ws and y must not be NULL");
  if (misaligned(ws, 4) || misaligned(bias, 4) || misaligned(y, y_dtype == 0 ? 4 : 2))
    return set_error(ERR_ALIGN, "scales and bias must be 4-byte aligned, y to its elements");
  if (ldy < (N > 1 ? M : 0)) return set_error(ERR_SHAPE, "ldy=%lld < M=%lld", (long long)ldy, (long long)M);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t need = qgemv_int8_linear_workspace_bytes(N, K);
  WorkspaceHold hold;
  if (workspace) {
    if (workspace_bytes < need)
      return set_error(ERR_ARG, "this call needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
    if (misaligned(workspace, 16)) return set_error(ERR_ALIGN, "workspace must be 16-byte aligned");
  } else if (int rc = own_workspace(st, need, &workspace, hold)) {
    return rc;
  }
  float* xs = static_cast<float*>(workspace);
  void* xq = static_cast<uint8_t*>(workspace) + (size_t)((N + 31) / 32 * 32) * 4;
  if (int rc = int8_quantize(x, dtype, ldx, N, K, xq, K, xs, st)) return rc;
  return int8_entry(xq, xs, K, wq, ws, ldw, bias, N, M, K, y, y_dtype, ldy, true, stream);
}

}  // extern "C"
