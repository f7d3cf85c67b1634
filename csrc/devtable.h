// Content-addressed, never-freed device copies of small launch tables.
//
// The grouped kernels (gradient gather, KL dot / apply, factor SYRK / EMA)
// used to take their job tables as ~1-4 KB by-value kernel arguments.  When
// such a launch is captured into a hipGraph and the graph is replayed
// back-to-back, the kernels read corrupted tables on ROCm 7.2 (garbage
// gathered gradients, a NaN / inf KL scale; scripts/probes/debug_replay_nan.py,
// profiles/README.md), while kernels that read their tables from device memory
// (the preconditioning GEMMs) replay correctly.  So every table now lives in
// device memory: a table seen before costs nothing (the same device copy is
// returned, so a captured graph and eager launches share an immutable table);
// a new one is copied from a pinned host copy that the cache owns forever.
//
// Whoever gets a table reads what was written.  An eager call's copy goes into
// its stream; until it is known to have ended, calls on other streams wait for
// it on the device.  In a capture the copy is made at once, on a stream of the
// cache's own that the host waits for: as a node of the graph it would leave the
// table unwritten for every eager call and other graph that comes before the
// first replay, and for good if the capture is given up.
#pragma once
#include "common.h"

#include <cstring>
#include <deque>
#include <mutex>
#include <string>
#include <unordered_map>
#include <vector>

namespace kfac_devtable {

struct Table {
  char *dev, *host;
  size_t bytes;
  bool written;             // its copy is known to have ended
  hipEvent_t copied;        // else: behind the copy, in the stream of the first call
};

struct Cache {
  std::mutex mu;
  std::unordered_map<std::string, Table> map;   // its elements stay where they are
  std::deque<Table*> pending;                   // not known to be written, first copy first
  std::vector<hipEvent_t> events;               // free ones
  hipStream_t own = nullptr;
  char* dev = nullptr;      // current device arena
  char* host = nullptr;     // matching pinned host arena
  size_t used = 0, cap = 0;
};

inline Cache& cache() {
  static Cache c;
  return c;
}

// Lets this thread make calls that a capture would forbid; none of them touches
// the capturing stream.
struct Relaxed {
  hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
  Relaxed() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
  ~Relaxed() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};

// the copy has been made when this returns, inside captures as well
inline hipError_t copy_now(Cache& c, const Table& t) {
  Relaxed relaxed;
  hipError_t e = hipSuccess;
  if (!c.own) e = hipStreamCreateWithFlags(&c.own, hipStreamNonBlocking);
  if (e == hipSuccess) e = hipMemcpyAsync(t.dev, t.host, t.bytes, hipMemcpyHostToDevice, c.own);
  if (e == hipSuccess) e = hipStreamSynchronize(c.own);
  return e;
}

// the copy is in `stream`, an event behind it
inline hipError_t copy_in(Cache& c, Table& t, hipStream_t stream) {
  hipError_t e = hipSuccess;
  if (c.events.empty()) {
    e = hipEventCreateWithFlags(&t.copied, hipEventDisableTiming);
  } else {
    t.copied = c.events.back();
    c.events.pop_back();
  }
  if (e == hipSuccess) e = hipMemcpyAsync(t.dev, t.host, t.bytes, hipMemcpyHostToDevice, stream);
  if (e == hipSuccess) e = hipEventRecord(t.copied, stream);
  return e;
}

// tables whose copies have ended
inline void settle(Cache& c) {
  Relaxed relaxed;
  while (!c.pending.empty()) {
    Table& t = *c.pending.front();
    if (!t.written && hipEventQuery(t.copied) != hipSuccess) {
      (void)hipGetLastError();               // not ready
      return;
    }
    t.written = true;
    c.events.push_back(t.copied);
    c.pending.pop_front();
  }
}

// Device pointer to an immutable copy of `bytes` bytes at `host`, written for
// whatever follows on `stream`.  Returns nullptr (and sets *err) on failure.
inline const void* get(const void* host, size_t bytes, hipStream_t stream, int* err) {
  Cache& c = cache();
  std::lock_guard<std::mutex> lk(c.mu);
  std::string key((const char*)host, bytes);
  auto it = c.map.find(key);
  if (it != c.map.end() && it->second.written) return it->second.dev;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  const bool capturing = hipStreamIsCapturing(stream, &cs) == hipSuccess &&
                         cs != hipStreamCaptureStatusNone;
  if (!capturing) settle(c);
  if (it != c.map.end()) {
    Table& t = it->second;
    hipError_t e = hipSuccess;
    if (!t.written) {
      // in a capture the same bytes once more: nothing in the graph can wait for the
      // other stream's copy
      e = capturing ? copy_now(c, t) : hipStreamWaitEvent(stream, t.copied, 0);
      if (e == hipSuccess && capturing) t.written = true;
    }
    if (e == hipSuccess) return t.dev;
    *err = (int)e;
    return nullptr;
  }
  const size_t need = (bytes + 255) / 256 * 256;
  // A new arena is not allocated inside a capture, so an eager call begins one
  // while the old one still has room for what a capture may bring (a training
  // step's tables: some 100 KB).
  const size_t reserve = (size_t)1 << 20;
  if (c.used + need + (capturing ? 0 : reserve) > c.cap) {
    const size_t cap = need + reserve > (size_t)(4 << 20) ? need + reserve : (size_t)(4 << 20);
    char* d = nullptr;
    char* h = nullptr;
    if (capturing) {
      *err = -20;   // would allocate inside a capture
      return nullptr;
    }
    Relaxed relaxed;          // another thread may be capturing
    if (hipMalloc(&d, cap) != hipSuccess || hipHostMalloc(&h, cap, 0) != hipSuccess) {
      (void)hipGetLastError();
      if (d) (void)hipFree(d);
      *err = -21;
      return nullptr;
    }
    c.dev = d; c.host = h; c.used = 0; c.cap = cap;
  }
  Table t = {c.dev + c.used, c.host + c.used, bytes, capturing, nullptr};
  c.used += need;
  memcpy(t.host, host, bytes);
  const hipError_t e = capturing ? copy_now(c, t) : copy_in(c, t, stream);
  if (e != hipSuccess) {
    *err = (int)e;
    return nullptr;
  }
  Table& kept = c.map.emplace(std::move(key), t).first->second;
  if (!capturing) c.pending.push_back(&kept);
  return kept.dev;
}

}  // namespace kfac_devtable
