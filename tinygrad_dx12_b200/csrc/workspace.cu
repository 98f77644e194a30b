// workspace.cu -- device memory that kernels leave partial results and tickets in, between a launch's CTAs.
//
// Calls on one stream follow one another, so they share a block per (kernel family, device, stream), allocated
// on the first call and kept for the life of the process. A recorded graph runs on whatever stream replays it,
// beside calls on the stream that recorded it and beside other recordings: the calls of a capture share a block
// of their own, which the graph owns (a user object) and which goes back to a list, for later recordings, when
// the graph and everything instantiated from it are gone. It is allocated outside the graph while that is being
// captured: a recorded step has no allocation nodes.
#include <map>
#include <mutex>
#include <tuple>
#include <vector>

#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

using Key = std::tuple<int, int, unsigned long long, unsigned long long>;  // kind, device, stream, capture (0: none)
struct Block {
  Key key;
  uint8_t *base;
  size_t zeroed;
};
struct State {
  std::mutex mutex;   // of the members below
  std::mutex making;  // one block is made at a time; never taken while `mutex` is held
  std::map<Key, Block *> used;
  std::vector<Block *> spare;  // of recordings that are gone
};
State &state() {  // never destroyed: graphs may outlive static objects
  static State *s = new State;
  return *s;
}

// Allocations of this thread are allowed while a stream is being captured: they are no part of the graph.
struct Relaxed {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// On a stream of its own, which neither waits for the caller's work nor becomes part of a capture.
cudaError_t zero(uint8_t *p, size_t n) {
  cudaStream_t s = nullptr;
  cudaError_t e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
  if (e != cudaSuccess) return e;
  e = cudaMemsetAsync(p, 0, n, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  cudaStreamDestroy(s);
  return e;
}

void CUDART_CB graph_is_gone(void *block) {  // no CUDA call may be made here
  Block *b = static_cast<Block *>(block);
  State &s = state();
  std::lock_guard<std::mutex> lock(s.mutex);
  auto it = s.used.find(b->key);
  if (it != s.used.end() && it->second == b) s.used.erase(it);
  s.spare.push_back(b);
}

}  // namespace

static int32_t find_or_make(WorkspaceKind kind, size_t bytes, size_t zeroed, cudaStream_t stream, uint8_t **base) {
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  unsigned long long id = (unsigned long long)(uintptr_t)stream, capture = 0;
  cudaGraph_t graph = nullptr;
  if (stream == cudaStreamLegacy) id = 0;
  if (stream == cudaStreamPerThread) B200_CUDA_TRY(cudaStreamGetId(stream, &id));  // one handle for every thread's
  if (id != 0) {  // the legacy stream cannot be captured
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    B200_CUDA_TRY(cudaStreamIsCapturing(stream, &cs));
    if (cs != cudaStreamCaptureStatusNone) {
      B200_CUDA_TRY(cudaStreamGetCaptureInfo_v2(stream, &cs, &capture, &graph, nullptr, nullptr));
      if (cs != cudaStreamCaptureStatusActive) return b200_set_error(B200_ERR_CUDA, "workspace: the stream's capture is invalid");
    }
  }
  const Key key(kind, dev, id, capture);
  State &s = state();
  auto found = [&]() {
    std::lock_guard<std::mutex> lock(s.mutex);
    auto it = s.used.find(key);
    if (it != s.used.end()) *base = it->second->base;
    return it != s.used.end();
  };
  if (found()) return B200_OK;
  std::lock_guard<std::mutex> making(s.making);
  if (found()) return B200_OK;
  Block *b = nullptr;
  if (capture != 0) {
    std::lock_guard<std::mutex> lock(s.mutex);
    for (size_t i = 0; i < s.spare.size() && b == nullptr; ++i)
      if (std::get<0>(s.spare[i]->key) == kind && std::get<1>(s.spare[i]->key) == dev) {
        b = s.spare[i];
        s.spare.erase(s.spare.begin() + i);
      }
  }
  Relaxed relaxed;
  if (b == nullptr) {
    b = new Block{key, nullptr, zeroed};
    const cudaError_t e = cudaMalloc((void **)&b->base, bytes);
    if (e != cudaSuccess) {
      delete b;
      cudaGetLastError();
      return b200_set_error(B200_ERR_CUDA, "workspace of %zu bytes: %s", bytes, cudaGetErrorString(e));
    }
  }
  b->key = key;
  cudaError_t e = zero(b->base, zeroed);
  if (e == cudaSuccess && capture != 0) {
    {
      std::lock_guard<std::mutex> lock(s.mutex);
      s.used[key] = b;
    }
    cudaUserObject_t object = nullptr;
    e = cudaUserObjectCreate(&object, b, graph_is_gone, 1, cudaUserObjectNoDestructorSync);
    if (e != cudaSuccess) {
      graph_is_gone(b);
    } else {
      e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
      if (e != cudaSuccess) cudaUserObjectRelease(object, 1);  // calls graph_is_gone
    }
  } else {
    std::lock_guard<std::mutex> lock(s.mutex);
    if (e == cudaSuccess) s.used[key] = b;
    else s.spare.push_back(b);
  }
  if (e != cudaSuccess) return b200_set_error(B200_ERR_CUDA, "workspace: %s", cudaGetErrorString(e));
  *base = b->base;
  return B200_OK;
}

int32_t workspace_of(WorkspaceKind kind, size_t bytes, size_t zeroed, cudaStream_t stream, uint8_t **base) {
  try {
    return find_or_make(kind, bytes, zeroed, stream, base);
  } catch (...) {
    return b200_set_error(B200_ERR_CUDA, "workspace: out of host memory");
  }
}

int32_t workspace_zero(WorkspaceKind kind) {
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  State &s = state();
  B200_CUDA_TRY(cudaDeviceSynchronize());
  std::lock_guard<std::mutex> making(s.making);
  std::lock_guard<std::mutex> lock(s.mutex);  // spare blocks are zeroed when they are handed out again
  for (auto &kv : s.used)
    if (std::get<0>(kv.first) == kind && std::get<1>(kv.first) == dev) B200_CUDA_TRY(zero(kv.second->base, kv.second->zeroed));
  return B200_OK;
}

}  // namespace b200
