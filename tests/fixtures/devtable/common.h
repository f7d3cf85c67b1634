// A HIP runtime that only keeps books, for csrc/devtable.h on the CPU: a stream's
// operations wait in its queue until the stream is run, those of a captured stream
// go into its graph, and a call that a capture forbids is counted.
#pragma once
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

struct FakeEvent {
  bool recorded = false, ended = false;
  struct FakeStream* on = nullptr;
};
struct FakeStream {
  std::vector<std::function<void()>> queue;
  std::vector<std::function<void()>>* graph = nullptr;      // where a capture puts them
};
typedef FakeStream* hipStream_t;
typedef FakeEvent* hipEvent_t;
enum hipError_t { hipSuccess = 0, hipErrorInvalid = 1, hipErrorNotReady = 600, hipErrorCapture = 900 };
enum hipStreamCaptureStatus { hipStreamCaptureStatusNone, hipStreamCaptureStatusActive };
enum hipStreamCaptureMode { hipStreamCaptureModeGlobal, hipStreamCaptureModeRelaxed };
enum hipMemcpyKind { hipMemcpyHostToDevice };
constexpr unsigned hipStreamNonBlocking = 1, hipEventDisableTiming = 2;

namespace fake {
inline int captures = 0, forbidden = 0, events = 0, copies = 0, allocations = 0;
inline hipStreamCaptureMode mode = hipStreamCaptureModeGlobal;
inline hipError_t unsafe() {
  if (captures && mode != hipStreamCaptureModeRelaxed) {
    ++forbidden;
    return hipErrorCapture;
  }
  return hipSuccess;
}
inline void put(hipStream_t s, std::function<void()> op) { (s->graph ? *s->graph : s->queue).push_back(op); }
inline void run(hipStream_t s) {
  std::vector<std::function<void()>> q;
  q.swap(s->queue);
  for (auto& op : q) op();
}
inline void begin(hipStream_t s, std::vector<std::function<void()>>* g) { s->graph = g; ++captures; }
inline void end(hipStream_t s) { s->graph = nullptr; --captures; }
inline void replay(std::vector<std::function<void()>>& g) { for (auto& op : g) op(); }
}  // namespace fake

inline hipError_t hipGetLastError() { return hipSuccess; }
inline hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus* st) {
  *st = s->graph ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
inline hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode* m) {
  const hipStreamCaptureMode old = fake::mode;
  fake::mode = *m;
  *m = old;
  return hipSuccess;
}
template <class T> hipError_t hipMalloc(T** p, size_t n) {
  if (const hipError_t e = fake::unsafe()) return e;
  ++fake::allocations;
  *p = (T*)memset(malloc(n), 0xAB, n);                    // nobody has written it
  return hipSuccess;
}
template <class T> hipError_t hipHostMalloc(T** p, size_t n, unsigned) {
  if (const hipError_t e = fake::unsafe()) return e;
  *p = (T*)malloc(n);
  return hipSuccess;
}
inline hipError_t hipFree(void* p) { free(p); return hipSuccess; }
inline hipError_t hipMemcpyAsync(void* d, const void* h, size_t n, hipMemcpyKind, hipStream_t s) {
  ++fake::copies;
  fake::put(s, [=] { memcpy(d, h, n); });
  return hipSuccess;
}
inline hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned flags) {
  if (const hipError_t e = fake::unsafe()) return e;
  if (flags != hipStreamNonBlocking) return hipErrorInvalid;
  *s = new FakeStream;
  return hipSuccess;
}
inline hipError_t hipStreamSynchronize(hipStream_t s) {
  if (const hipError_t e = fake::unsafe()) return e;
  if (s->graph) return hipErrorCapture;
  fake::run(s);
  return hipSuccess;
}
inline hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
  if (const hipError_t err = fake::unsafe()) return err;
  ++fake::events;
  *e = new FakeEvent;
  return hipSuccess;
}
inline hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) {
  if (s->graph) return hipErrorCapture;
  e->recorded = true;
  e->ended = false;
  e->on = s;
  fake::put(s, [=] { e->ended = true; });
  return hipSuccess;
}
inline hipError_t hipEventQuery(hipEvent_t e) {
  if (const hipError_t err = fake::unsafe()) return err;
  return e->ended ? hipSuccess : hipErrorNotReady;
}
inline hipError_t hipStreamWaitEvent(hipStream_t s, hipEvent_t e, unsigned) {
  if (s->graph || !e->recorded) return hipErrorCapture;
  if (s != e->on) fake::put(s, [=] { if (!e->ended) fake::run(e->on); });
  return hipSuccess;
}
