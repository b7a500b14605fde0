// operators_abi.h -- what the entry points of the op-level operators share
// (operators.hip, cache.hip): the guard against exceptions, refusals, handles, and
// whether operands meet in memory.
#pragma once

#include "runtime.h"

#include <cstdio>
#include <new>

namespace tgohip {

// Entry points do not throw across the C ABI, and a refused call leaves no error behind
// that the next launch would report as its own.
template <typename F>
int guarded(F f) {
  try {
    const int rc = f();
    if (rc) (void)hipGetLastError();
    return rc;
  } catch (const std::bad_alloc&) {
    return fail(TGOHIP_ENOMEM, "host allocation failed");
  } catch (const std::exception& e) {
    return fail(TGOHIP_EDEVICE, std::string("internal: ") + e.what());
  }
}

// Makes the context's device current for a call, and the caller's again after it.
struct OnDevice {
  int prev = -1;
  bool moved = false;
  explicit OnDevice(int device) {
    if (hipGetDevice(&prev) == hipSuccess && prev != device) moved = hipSetDevice(device) == hipSuccess;
  }
  ~OnDevice() {
    if (moved) (void)hipSetDevice(prev);
  }
};

inline int refuse(const std::string& why) { return fail(TGOHIP_EINVAL, why); }
inline int no_ctx(const char* what) { return refuse(std::string(what) + ": the context is missing"); }

// Making, changing or freeing a handle copies, allocates and waits, which a graph
// cannot hold.
inline int no_capture(tgohip_ctx* c, const char* what) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  const hipError_t e = hipStreamIsCapturing(c->stream, &st);
  if (e != hipSuccess) return fail(TGOHIP_EDEVICE, hip_message(e, what));
  if (st == hipStreamCaptureStatusNone) return 0;
  return fail(TGOHIP_ESTATE, std::string(what) + ": the context's stream is being captured");
}

template <typename T>
T* find(std::map<int, T>& m, int handle, const char* what) {
  auto it = m.find(handle);
  if (it != m.end()) return &it->second;
  refuse(std::string(what) + ": no handle " + std::to_string(handle));
  return nullptr;
}

inline bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }
inline int64_t elt(int f16) { return f16 ? 2 : 4; }

// A device operand: `rows` rows of `heads` heads of d elements, strides in bytes.
struct Span {
  const char* p;
  int64_t rows, heads, row, head, d;
  int64_t width() const { return (heads - 1) * head + d; }  // of one row
  int64_t end() const { return rows ? (rows - 1) * row + width() : 0; }
};
// Whether two operands may share memory: apart, or columns of the same rows that
// do not meet.
inline bool meet(const Span& a, const Span& b) {
  if (!a.rows || !b.rows) return false;
  if (a.p + a.end() <= b.p || b.p + b.end() <= a.p) return false;
  if (a.row == b.row && a.row > 0 && a.width() <= a.row && b.width() <= a.row) {
    int64_t off = (b.p - a.p) % a.row;
    if (off < 0) off += a.row;
    if (off >= a.width() && off + b.width() <= a.row) return false;
  }
  return true;
}
inline bool same(const Span& a, const Span& b) {
  return a.p == b.p && a.d == b.d && (a.rows <= 1 || a.row == b.row) && (a.heads <= 1 || a.head == b.head);
}

inline std::string num(double v) {
  char b[64];
  snprintf(b, sizeof b, "%g", v);
  return b;
}

}  // namespace tgohip
