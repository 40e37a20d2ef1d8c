"""The C ABI's per-stream workspace (csrc/capi.cu) under host threads, on the CPU:
its functions are compiled as they stand in the source against a stand-in for the
CUDA runtime.  A call keeps its stream's buffer until its launches are enqueued:
another thread's call on the stream waits, and does not free the buffer to grow it."""

import os
import re
import shutil
import subprocess

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "qgemv_roofline_b200", "csrc", "capi.cu")

HARNESS = r"""
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <thread>
#include <tuple>
#include <utility>

typedef struct Stream* cudaStream_t;
typedef int cudaError_t;
enum { cudaSuccess = 0 };
enum cudaStreamCaptureStatus { cudaStreamCaptureStatusNone = 0 };
#define cudaStreamPerThread ((cudaStream_t)2)
static std::atomic<void*> last_freed{nullptr};
cudaError_t cudaGetDevice(int* d) { *d = 0; return 0; }
cudaError_t cudaSetDevice(int) { return 0; }
cudaError_t cudaDeviceSynchronize() { return 0; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return 0; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) { *s = cudaStreamCaptureStatusNone; return 0; }
cudaError_t cudaMalloc(void** p, size_t n) { *p = malloc(n); return 0; }
cudaError_t cudaFree(void* p) { last_freed = p; return 0; }  // kept: an address is never given twice
const char* cudaGetErrorString(cudaError_t) { return ""; }
enum { OK = 0, ERR_CUDA = 4, ERR_UNSUPPORTED = 5 };
int set_error(int code, const char*, ...) { return code; }
using WorkspaceHold = std::unique_lock<std::mutex>;
int stream_workspace(cudaStream_t st, size_t bytes, void** out, WorkspaceHold& hold);
int release_workspaces();
namespace {
@SOURCE@

#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main() {
  const cudaStream_t st = (cudaStream_t)64, other = (cudaStream_t)128;
  void *a = nullptr, *b = nullptr, *c = nullptr;
  {
    WorkspaceHold mine;
    CHECK(stream_workspace(st, 1000, &a, mine) == OK && mine.owns_lock());
    // another stream's call does not wait
    std::thread([&] { WorkspaceHold h; stream_workspace(other, 10, &c, h); }).join();
    CHECK(c && c != a);
    std::atomic<bool> has{false}, released{false};
    std::thread t([&] {
      WorkspaceHold h;
      stream_workspace(st, 1 << 20, &b, h);  // larger: the old buffer goes
      has = true;
    });
    std::thread r([&] { release_workspaces(); released = true; });
    std::this_thread::sleep_for(std::chrono::milliseconds(200));
    CHECK(!has && !released && last_freed.load() != a);
    mine.unlock();  // the launches are enqueued
    t.join();
    r.join();
    CHECK(has && released);
  }
  {
    WorkspaceHold h;
    CHECK(stream_workspace(st, 16, &a, h) == OK);
  }
  {
    WorkspaceHold h;
    CHECK(stream_workspace(st, 16, &b, h) == OK && a == b);  // kept from call to call
  }
  // the per-thread default stream: a buffer for each thread
  {
    WorkspaceHold h;
    CHECK(stream_workspace(cudaStreamPerThread, 16, &a, h) == OK);
    std::thread([&] { WorkspaceHold g; stream_workspace(cudaStreamPerThread, 16, &b, g); }).join();
    CHECK(a != b);
  }
  CHECK(release_workspaces() == OK);
  return 0;
}
"""


def functions():
    with open(SOURCE) as f:
        text = f.read()
    start = re.search(r"^(struct StreamWorkspace|std::mutex g_ws_mu)", text, re.M).start()
    return text[start:text.index("namespace {", start)]


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_a_call_keeps_the_workspace_until_its_launches_are_enqueued(tmp_path):
    src = tmp_path / "ws.cpp"
    src.write_text(HARNESS.replace("@SOURCE@", functions()))
    exe = str(tmp_path / "ws")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", str(src), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_every_user_of_the_workspace_holds_it():
    with open(SOURCE) as f:
        text = f.read()
    calls = re.findall(r"\b(?:stream|own)_workspace\(([^;{]*?)\)\) \{", text)
    assert len(calls) == 5 and all(c.endswith(", hold") for c in calls), calls
