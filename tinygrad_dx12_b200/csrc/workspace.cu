// workspace.cu -- device memory that kernels leave partial results and tickets in, between a launch's CTAs.
//
// Calls on one stream follow one another, so they share a block per (kernel family, device, stream), allocated
// on the first call and kept for the life of the process. A recorded graph runs on whatever stream replays it,
// beside calls on the stream that recorded it and beside other recordings: the calls of a capture share a block
// of their own, until whoever holds the graph says that it is gone (b200_capture_release); then it serves a later
// capture. It is allocated outside the graph while that is being captured: a recorded step has no allocation
// nodes. (A user object, by which the graph would say so itself, costs 2 to 3 us of every replay.)
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
  size_t bytes, tickets;
};
struct State {
  std::mutex mutex;   // of the members below
  std::mutex making;  // one block is made at a time; never taken while `mutex` is held
  std::map<Key, Block *> used;
  std::vector<Block *> spare;  // of recordings that are gone; their tickets are zero, as kernels leave them
};
State &state() {  // never destroyed: a recording may be released after static objects
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

// The capture that `stream` is in, 0 if none.
int32_t capture_of(cudaStream_t stream, unsigned long long *id) {
  *id = 0;
  if (stream == nullptr || stream == cudaStreamLegacy) return B200_OK;  // cannot be captured
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  B200_CUDA_TRY(cudaStreamIsCapturing(stream, &cs));
  if (cs == cudaStreamCaptureStatusNone) return B200_OK;
  B200_CUDA_TRY(cudaStreamGetCaptureInfo_v2(stream, &cs, id, nullptr, nullptr, nullptr));
  if (cs != cudaStreamCaptureStatusActive) return b200_set_error(B200_ERR_CUDA, "the stream's capture is invalid");
  return B200_OK;
}

}  // namespace

static int32_t find_or_make(WorkspaceKind kind, size_t bytes, size_t tickets, cudaStream_t stream, uint8_t **base) {
  int dev = 0;
  B200_CUDA_TRY(cudaGetDevice(&dev));
  unsigned long long id = (unsigned long long)(uintptr_t)stream, capture = 0;
  if (stream == cudaStreamLegacy) id = 0;
  if (stream == cudaStreamPerThread) B200_CUDA_TRY(cudaStreamGetId(stream, &id));  // one handle for every thread's
  if (int32_t rc = capture_of(stream, &capture)) return rc;
  const Key key(kind, dev, id, capture);
  State &s = state();
  auto found = [&](bool spare) {
    std::lock_guard<std::mutex> lock(s.mutex);
    auto it = s.used.find(key);
    if (it == s.used.end() && spare)
      for (size_t i = 0; i < s.spare.size(); ++i)
        if (std::get<0>(s.spare[i]->key) == kind && std::get<1>(s.spare[i]->key) == dev) {
          s.spare[i]->key = key;
          it = s.used.emplace(key, s.spare[i]).first;
          s.spare.erase(s.spare.begin() + i);
          break;
        }
    if (it != s.used.end()) *base = it->second->base;
    return it != s.used.end();
  };
  if (found(false)) return B200_OK;
  std::lock_guard<std::mutex> making(s.making);
  if (found(capture != 0)) return B200_OK;
  Relaxed relaxed;
  uint8_t *p = nullptr;
  cudaError_t e = cudaMalloc((void **)&p, bytes + tickets);
  if (e == cudaSuccess && tickets > 0) e = zero(p + bytes, tickets);
  if (e != cudaSuccess) {
    cudaGetLastError();
    if (p != nullptr) cudaFree(p);
    return b200_set_error(B200_ERR_CUDA, "workspace of %zu bytes: %s", bytes + tickets, cudaGetErrorString(e));
  }
  std::lock_guard<std::mutex> lock(s.mutex);
  s.used[key] = new Block{key, p, bytes, tickets};
  *base = p;
  return B200_OK;
}

int32_t workspace_of(WorkspaceKind kind, size_t bytes, size_t tickets, cudaStream_t stream, uint8_t **base) {
  try {
    return find_or_make(kind, bytes, tickets, stream, base);
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
  std::lock_guard<std::mutex> lock(s.mutex);
  std::vector<Block *> all(s.spare);
  for (auto &kv : s.used) all.push_back(kv.second);
  for (Block *b : all)
    if (std::get<0>(b->key) == kind && std::get<1>(b->key) == dev) B200_CUDA_TRY(zero(b->base + b->bytes, b->tickets));
  return B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" {

int32_t b200_capture_id(void *stream, uint64_t *id) {
  if (id == nullptr) return b200_set_error(B200_ERR_INVALID, "capture_id: null pointer");
  unsigned long long c = 0;
  if (int32_t rc = capture_of((cudaStream_t)stream, &c)) return rc;
  *id = c;
  return B200_OK;
}

int32_t b200_capture_release(uint64_t id) {
  if (id == 0) return B200_OK;
  try {
    State &s = state();
    std::lock_guard<std::mutex> lock(s.mutex);
    for (auto it = s.used.begin(); it != s.used.end();) {
      if (std::get<3>(it->first) == id) {
        s.spare.push_back(it->second);
        it = s.used.erase(it);
      } else {
        ++it;
      }
    }
  } catch (...) {
    return b200_set_error(B200_ERR_CUDA, "capture_release: out of host memory");
  }
  return B200_OK;
}

}  // extern "C"
